// lm_loss.cu - cross entropy of rows h [M][K] under a head w [V][K], and its gradient, without the logits in memory.
//
//   z = scale h w^T,  loss_i = log sum_j exp z_ij - z_i,target        P = softmax(z) - onehot,  dh_i = scale g_i P_i w,  dw = P^T (scale g h)
//
// Forward: one product whose epilogue keeps of a 256 x 256 tile of logits, per row, the largest one, the sum of the exponentials below it and the target's, all in fp32;
// a second kernel joins the tiles of a row.  Backward: the vocabulary goes in pieces.  The product is taken again for a piece, its epilogue turns logits into P (bf16, a
// piece of at most 128 MB or 4096 columns, about what L2 holds), and two products take P to dh (fp32 sums over the pieces) and to the piece's rows of dw; their tiles are dealt
// to the pairs together.  (8192 x 32768 x 2048 and 4096 x 65536 x 1024, loss and gradients, ms, pieces of 32, 64, 128 and 256 MB: 4.55 and 1.97, 3.58 and 1.90, 3.50 and 1.80,
// 3.52 and 1.85.)
//
// What is rounded to fewer than 32 bits.  P, to bf16: as an operand of the tensor cores; in two terms the three products would take 12 M V K operations, not 8, for results that are
// bf16 themselves.  It is rounded without g: 1 - p of a row's target, which is most of its gradient, then lies just below a power of two where steps are fine, and the roundings of
// the rows do not go one way (8192 rows: 1.7e-3 to 1.9e-3 of the gradients' norm, of which the results' own rounding is 1.66e-3; with g inside 3.0e-3).  One g for all rows
// multiplies the sums; rows with their own take it into h for dw, rounded once more by half a step of bf16 (it belongs inside that contraction), and behind the sums for dh.  fp32
// rows of the forward pass are three bf16 terms, 24 bits; their losses are 8.4e-7 off where elementary fp32 operations are 2.9e-7 off (the tensor core's sums are cut off, not rounded).
//
// All of them are one kernel on pairs of SMs: a cluster of two CTAs owns a 256 x 256 tile, tcgen05.mma (cta_group::2) multiplies the 256 rows of both by the 256 columns of
// both, and the accumulators (two per CTA: a tile is taken out while the next is multiplied) live in tensor memory.
//   warp 0    one lane per CTA: TMA loads of its halves into a ring of stages; every byte of both CTAs counts on the leader's barrier
//   warp 1    leader only: one elected lane issues the pair's MMAs, commits to the barriers of both CTAs
//   warps 2-9 epilogue of the CTA's 128 rows, half of the columns each
// P w contracts over rows of w and P^T h over rows of both: those operands lie with the contraction along their rows in memory, and the MMA takes them so
// (MN-major descriptors); nothing is transposed.
#include <algorithm>

#include <cuda_bf16.h>

#include "attention_split.h"
#include "engine_internal.h"
#include "gemm_tcgen05.h"
#include "lm_loss.h"
#include "lm_mxfp4.h"
#include "lm_store.cuh"
#include "tensor_cores.cuh"

namespace lm {
namespace {

using namespace dia;

enum Kind { kStats, kProbs, kGrads };

constexpr int kTileN = 256, kBK = 64, kTileBytes = 128 * kBK * 2;          // 16 KB: 128 rows of an operand, 64 of the contraction
constexpr int kWarps = 8, kThreads = 64 + 32 * kWarps, kStagesMost = 6, kTurn = kWarps * 4096;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// (PAIR: see loss_product_kernel)
template <int TERMS, bool PAIR>
struct Ring {
    static constexpr int kStage = (TERMS + (PAIR ? 1 : 2)) * kTileBytes, kStages = TERMS == 1 ? (PAIR ? 6 : 4) : PAIR ? 3 : 2;
    static constexpr int kSmem = kStages * kStage + kTurn + 1024 + 256;
};

// k-blocks of an accumulator.  The tensor core cuts its sum off at every step of 16, by up to 2^-23 of it, so that a sum of terms of one sign drifts towards zero.  The losses'
// logits: 1024 products of one term, 512 of three (64 and 96 steps: 2^-16 of them).  Of P, which is rounded to bf16 behind, 4096 channels (256 steps: 2^-15 of a logit), and of the
// gradients, whose results are bf16, 32768 rows or columns (2048 steps: 2^-12 of the sum, a sixteenth of that rounding).  What is longer is summed in fp32.
template <int KIND, int TERMS>
constexpr int kChunkOf = KIND == kStats ? (TERMS == 1 ? 16 : 8) : KIND == kProbs ? 64 : 512;
constexpr int kSumsCtas = 148, kSumsFloats = 128 * kTileN;      // sums of the pieces that came before the last one: CTAs that have room for them, numbers of each

// Tiles of one product, and what they are made of (kGrads has two products)
struct Tiles {
    int M, N, K;                     // rows and columns of the product, length of the contraction
    int rows;                        // of a tile: 256, or 128 on one SM
    int splits;                      // pairs that share the contraction of a tile
    __host__ __device__ int tiles_m() const { return (M + rows - 1) / rows; }
    __host__ __device__ int tiles_n() const { return (N + kTileN - 1) / kTileN; }
    __host__ __device__ long long tiles() const { return N > 0 ? (long long)tiles_m() * tiles_n() * splits : 0; }
    __host__ __device__ int blocks() const { return (K + kBK - 1) / kBK; }
    __host__ __device__ int share() const { return (blocks() + splits - 1) / splits; }
};

struct LossTiles {
    Tiles own;                       // kStats, kProbs: the logits; kGrads: dh
    Tiles head;                      // kGrads: dw
    int first_head, many, extra;     // kGrads: whether dw's tiles are the longer ones, which go first; tiles of the longer kind; the shorter ones as long as one of them
    const void* targets; int targets64; long long ignore;
    float c;                         // scale log2(e)
    unsigned* arrived;               // kStats: set to zero for the kernel that joins the tiles
    float2* part; float* hit;        // kStats: [M][2 column tiles] largest c z and sum of 2^(c z - it); [M] z of the target
    const float2* kept; int v0, V;   // kProbs: [M] lse and loss; columns v0 .. of the head
    __nv_bfloat16* p; int ldp;
    float* acc; int ld_acc, add;     // kGrads, dh: [splits][M][ld_acc]; add: to what is there
    __nv_bfloat16* out; int wide;    // dw: [M][N]; wide: 16-byte stores
    float* sums;                     // kProbs, dw: [CTA][kSumsFloats] where an accumulator does not take the whole contraction
    const float *grad, *count; float scale;        // dw: what the sums are multiplied by (grad null: nothing)
    int* ran_out;
    unsigned polls;
};

__device__ __forceinline__ long long target_of(const void* t, int wide, int i) {
    return wide ? reinterpret_cast<const long long*>(t)[i] : (long long)reinterpret_cast<const int*>(t)[i];
}

// An operand whose contraction lies along memory rows: [64 k][64 channels] boxes of 128-byte rows with the 128-byte swizzle.  Eight rows of k are 1024 bytes apart
// (stride byte offset), 64 channels further the next box begins, 8192 bytes on (leading byte offset).
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t smem_addr) {
    const uint32_t lo = ((smem_addr & 0x3FFFFu) >> 4) | ((8192u >> 4) << 16);
    const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 32 rows x 128 columns of bf16, of which this warp has half the columns (lane = row), by the two warps of a quarter to out [..][ld] from (row0, c0) on, `rows` and `cols` of them
__device__ __forceinline__ void store_128(unsigned char* panel, const uint32_t (&y)[32], __nv_bfloat16* out, long long ld, long long row0, int rows, int c0, int cols, bool wide,
                                          int quarter, int half, int lane) {
    fill_panel(panel, half, y, lane);
    panel_sync(quarter);
    store_panel<2>(panel, reinterpret_cast<char*>(out + row0 * ld + c0), (size_t)ld * 2, half, rows, min(cols, 128), wide, lane);
    panel_sync(quarter);
}

struct Tile {
    bool head;
    int m, n, share, kb0, kb1;       // row and column block, share of the contraction and its k-blocks
};
// Tile k of a pair, false behind its last one.  Longer tiles are dealt first, one a round; the pairs that a last, partial round of them leaves out get `extra` shorter ones in
// its place, the rest goes in rounds.  (One kind: pair, pair + pairs, ..)
__device__ __forceinline__ bool tile_of(const LossTiles& p, int pair, int pairs, int k, Tile& t) {
    const int all = (int)(p.own.tiles() + p.head.tiles()), few = all - p.many, left = p.many % pairs, rounds = (p.many - pair + pairs - 1) / pairs;
    int i;
    if (pair < p.many && k < rounds) {
        i = pair + k * pairs;
    } else {
        k -= pair < p.many ? rounds : 0;
        const int more = left ? p.extra : 0;
        if (left && pair >= left && k < more) {
            i = k * (pairs - left) + pair - left;
        } else {
            if (left && pair >= left) k -= more;
            i = more * (pairs - left) + k * pairs + (pair - left + pairs) % pairs;
        }
        if (i >= few) return false;
        i += p.many;
    }
    t.head = (i < p.many) == (p.first_head != 0);
    if (i >= p.many) i -= p.many;
    const Tiles& of = t.head ? p.head : p.own;
    const int tm = of.tiles_m(), tn = of.tiles_n();
    t.m = i % tm;
    t.n = i / tm % tn;
    t.share = i / (tm * tn);
    t.kb0 = t.share * of.share();
    t.kb1 = min(t.kb0 + of.share(), of.blocks());
    return true;
}

// PAIR false: one SM per 128 x 256 tile, for 128 rows and less, half of whose pair would multiply nothing (losses of 64 rows x 32768 x 2048, us, pairs / one SM: bf16
// 37 / 32, fp32 rows 72 / 47; 131072 x 4096 bf16 233 / 199).
template <int KIND, int TERMS, bool PAIR = true>
__global__ void __cluster_dims__(PAIR ? 2 : 1, 1, 1) __launch_bounds__(kThreads, 1)
loss_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_ha,
                    const __grid_constant__ CUtensorMap map_hb, const __grid_constant__ LossTiles p) {
    constexpr int kStage = Ring<TERMS, PAIR>::kStage, kStages = Ring<TERMS, PAIR>::kStages, kChunk = kChunkOf<KIND, TERMS>;
    static_assert(PAIR || KIND != kGrads, "both gradients go on pairs");
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* turn = smem + kStages * kStage;
    uint64_t* full = reinterpret_cast<uint64_t*>(turn + kTurn);              // (the leader's alone)
    uint64_t* empty = full + kStagesMost;
    uint64_t* t_full = empty + kStagesMost;
    uint64_t* t_empty = t_full + 2;                                          // (the leader's alone)
    PairEnd* end = reinterpret_cast<PairEnd*>(t_empty + 2);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(end + 1);
    static_assert((2 * kStagesMost + 4) * 8 + sizeof(PairEnd) + 4 <= 256, "barrier region");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? blockIdx.x & 1 : 0;
    const int pair = PAIR ? blockIdx.x >> 1 : blockIdx.x, pairs = PAIR ? gridDim.x >> 1 : gridDim.x;
    const auto everyone = [] {
        if constexpr (PAIR) cluster_sync_all();
        else __syncthreads();
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&t_full[i], 1); mbar_init(&t_empty[i], (PAIR ? 2 : 1) * kWarps); }
        pair_begin(end);
        fence_mbar_init();
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    everyone();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;
    // Launched while the predecessor may still run.  Tensor memory is held while this waits for it, but an SM has no room for this kernel beside another one that takes some; the
    // successor may come as soon as every CTA has its own.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (KIND == kStats && blockIdx.x == 0 && threadIdx.x == 0) *p.arrived = 0u;
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            unsigned i = 0;
            Tile t;
            for (int n = 0; ok && tile_of(p, pair, pairs, n, t); ++n) {
                const int a0 = t.m * (PAIR ? 256 : 128) + (int)rank * 128, b0 = t.n * kTileN + (int)rank * 128;
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++i) {
                    const unsigned s = i % kStages;
                    if (!lane_wait(&empty[s], ((i / kStages) & 1u) ^ 1u, p.polls)) { ok = false; break; }
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], (PAIR ? 2u : 1u) * kStage);
                    const uint32_t bar = at_rank(&full[s], 0), dst = smem_u32(smem + s * kStage), k = kb * kBK;
                    if constexpr (KIND == kGrads) {
                        if (t.head) {
                            tma_load_2d_pair(dst, &map_ha, bar, a0, k);
                            tma_load_2d_pair(dst + kTileBytes / 2, &map_ha, bar, a0 + 64, k);
                            tma_load_2d_pair(dst + kTileBytes, &map_hb, bar, b0, k);
                            tma_load_2d_pair(dst + kTileBytes + kTileBytes / 2, &map_hb, bar, b0 + 64, k);
                        } else {                              // (of the head the piece's rows)
                            tma_load_2d_pair(dst, &map_a, bar, k, a0);
                            tma_load_2d_pair(dst + kTileBytes, &map_b, bar, b0, p.v0 + k);
                            tma_load_2d_pair(dst + kTileBytes + kTileBytes / 2, &map_b, bar, b0 + 64, p.v0 + k);
                        }
                    } else if constexpr (!PAIR) {
                        tma_load_2d(dst + TERMS * kTileBytes, &map_b, bar, k, p.v0 + b0);
                        tma_load_2d(dst + (TERMS + 1) * kTileBytes, &map_b, bar, k, p.v0 + b0 + 128);
#pragma unroll
                        for (int tm = 0; tm < TERMS; ++tm) tma_load_2d(dst + tm * kTileBytes, &map_a, bar, k, tm * p.own.M + a0);
                    } else {
                        tma_load_2d_pair(dst + TERMS * kTileBytes, &map_b, bar, k, p.v0 + b0);
#pragma unroll
                        for (int tm = 0; tm < TERMS; ++tm) tma_load_2d_pair(dst + tm * kTileBytes, &map_a, bar, k, tm * p.own.M + a0);
                    }
                }
            }
            // (the leader's last commits arrive here: not after this CTA has gone)
            for (unsigned j = i > (unsigned)kStages ? i - kStages : 0; j < i && ok; ++j) ok = lane_wait(&empty[j % kStages], (j / kStages) & 1u, p.polls);
            if constexpr (PAIR) pair_issued(end, rank, i);
            else copies_landed(full, kStages, i);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            unsigned i = 0, it = 0;                           // k-blocks and uses of an accumulator so far
            Tile t;
            for (int n = 0; ok && tile_of(p, pair, pairs, n, t); ++n) {
                const bool a_mn = KIND == kGrads && t.head, b_mn = KIND == kGrads;
                // fp32 accumulators, bf16 operands, which of them are MN-major, N = 256, M = 256 or 128
                const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(kTileN >> 3) << 17) | ((PAIR ? 16u : 8u) << 24);
                const uint32_t a_step = a_mn ? 2048 >> 4 : 2, b_step = b_mn ? 2048 >> 4 : 2;        // 16 of the contraction, in descriptor units
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++i) {
                    const bool first = (kb - t.kb0) % kChunk == 0, last = kb == t.kb1 - 1 || (kb - t.kb0) % kChunk == kChunk - 1;
                    if (first) {
                        if (!pair_wait(&t_empty[it & 1u], ((it >> 1) & 1u) ^ 1u, p.polls)) { ok = false; break; }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    }
                    const uint32_t d = tmem_base + (it & 1u) * kTileN;
                    const unsigned s = i % kStages;
                    if (!pair_wait(&full[s], (i / kStages) & 1u, p.polls)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = smem_u32(smem + s * kStage);
                    const uint64_t bdesc = b_mn ? umma_desc_mn(at + TERMS * kTileBytes) : umma_desc(at + TERMS * kTileBytes);
                    if (elect_one_sync()) {
#pragma unroll
                        for (int u = 0; u < TERMS; ++u) {
                            const uint32_t a_at = at + (TERMS - 1 - u) * kTileBytes;                 // the smallest term first
                            const uint64_t adesc = a_mn ? umma_desc_mn(a_at) : umma_desc(a_at);
#pragma unroll
                            for (int j = 0; j < kBK / 16; ++j) {
                                const uint32_t more = (u | j) != 0 || !first ? 1u : 0u;
                                if constexpr (PAIR) umma_bf16_pair(d, adesc + a_step * j, bdesc + b_step * j, idesc, more);
                                else umma_bf16(d, adesc + a_step * j, bdesc + b_step * j, idesc, more);
                            }
                        }
                        if constexpr (PAIR) {
                            umma_commit_pair(&empty[s]);
                            if (last) umma_commit_pair(&t_full[it & 1u]);
                        } else {
                            umma_commit(&empty[s]);
                            if (last) umma_commit(&t_full[it & 1u]);
                        }
                    }
                    __syncwarp();
                    if (last) ++it;
                }
            }
            mmas_ended<PAIR>(&end->done);
        }
    } else {
        const int q = warp & 3, c_half = (warp - 2) >> 2 << 7;               // (a warp reads the 32 lanes of its number mod 4) and its half of the columns
        const int half = (warp - 2) >> 2;
        unsigned char* const panel = turn + q * kPanelBytes;                 // of both warps that read these lanes; blk: this one's share of it
        unsigned char* const blk = panel + half * 4096;
        float factor = 1.f;
        if (KIND == kGrads && p.grad) {
            factor = *p.grad * p.scale;
            if (p.count) factor /= fmaxf(*p.count, 1.f);
        }
        unsigned it = 0;
        // this warp has read the accumulator (relaxed: a release would wait for the warp's stores to be seen, whose addresses the MMAs have nothing to do with)
        const auto taken = [&]() {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(at_rank(&t_empty[it & 1u], 0)) : "memory");
            ++it;
        };
        Tile t;
        for (int tile = 0; tile_of(p, pair, pairs, tile, t); ++tile) {
            const Tiles& of = KIND == kGrads && t.head ? p.head : p.own;
            const int n0 = t.n * kTileN + c_half, row0 = t.m * (PAIR ? 256 : 128) + (int)rank * 128 + q * 32, rows = min(32, of.M - row0), row = row0 + lane;
            const bool mine = row < of.M;
            const auto tile_at = [&]() { return tmem_base + ((uint32_t)(q * 32) << 16) + (it & 1u) * kTileN; };
            const auto from = [&]() { return tile_at() + c_half; };
            const auto wait = [&]() {
                ok = ok && pair_wait(&t_full[it & 1u], (it >> 1) & 1u, p.polls);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            };
            // A contraction longer than an accumulator's: the pieces before the last one, added in this thread's own place; what came before columns 32 j .. of the warp's (of the
            // two times 64 that it stores) is then added to the last piece.
            const int chunks = (t.kb1 - t.kb0 + kChunk - 1) / kChunk;
            float* const sums = p.sums + (size_t)blockIdx.x * kSumsFloats + (threadIdx.x - 64);
            const auto add_earlier = [&](uint32_t (&v)[32], int j) {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + sums[(j * 32 + e) * 32 * kWarps]);
            };
            const auto earlier = [&]() {
#pragma unroll 1
                for (int c = 0; c + 1 < chunks; ++c) {
                    wait();
#pragma unroll 1
                    for (int j = 0; j < 4; ++j) {
                        uint32_t v[32];
                        tmem_columns32(tile_at() + (j >> 1) * 128 + half * 64 + (j & 1) * 32, v);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        if (c) add_earlier(v, j);
#pragma unroll
                        for (int e = 0; e < 32; ++e) sums[(j * 32 + e) * 32 * kWarps] = __uint_as_float(v[e]);
                    }
                    taken();
                }
            };
            if constexpr (KIND == kStats) {
                const long long target = mine ? target_of(p.targets, p.targets64, row) : -1;
                // (the pieces meet in registers)
                float z[128];
#pragma unroll
                for (int e = 0; e < 128; ++e) z[e] = 0.f;
                for (int kb = 0; kb < of.blocks(); kb += kChunk) {
                    wait();
#pragma unroll
                    for (int cb = 0; cb < 4; ++cb) {
                        uint32_t v[32];
                        tmem_columns32(from() + cb * 32, v);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int e = 0; e < 32; ++e) z[cb * 32 + e] += __uint_as_float(v[e]);
                    }
                    taken();
                }
                if (mine && target >= n0 && target < n0 + 128 && target < of.N) {
                    float at = 0.f;
#pragma unroll
                    for (int e = 0; e < 128; ++e) at = target == n0 + e ? z[e] : at;
                    p.hit[row] = ok ? at : CUDART_NAN_F;
                }
                if (n0 + 128 > of.N) {
#pragma unroll
                    for (int e = 0; e < 128; ++e) if (n0 + e >= of.N) z[e] = -CUDART_INF_F;
                }
                float top[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F}, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 128; ++e) top[e & 3] = fmaxf(top[e & 3], z[e]);
                const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.c;
                const float below = most == -CUDART_INF_F ? 0.f : most;              // (nothing but minus infinities)
#pragma unroll
                for (int e = 0; e < 128; ++e) sum[e & 3] += exp2_fast(fmaf(z[e], p.c, -below));
                if (mine)
                    p.part[(size_t)row * (2 * of.tiles_n()) + 2 * t.n + (c_half >> 7)] =
                        ok ? make_float2(most, (sum[0] + sum[1]) + (sum[2] + sum[3])) : make_float2(CUDART_NAN_F, CUDART_NAN_F);      // (no result)
            } else if constexpr (KIND == kProbs) {
                // rows that do not count are zeros, whatever they hold; one with a target that is not there NaN
                float base = 0.f, own = 0.f;
                int target = -1;
                bool counts = false;
                if (mine) {
                    const long long to = target_of(p.targets, p.targets64, row);
                    counts = to != p.ignore;
                    const float2 kept = p.kept[row];
                    const bool there = to >= 0 && to < p.V;
                    base = there ? kept.x * kLog2e : CUDART_NAN_F;
                    own = expm1f(-kept.y);                    // p - 1 of the target: keeps its digits where p is next to one
                    if (there) target = (int)to - p.v0;
                }
                earlier();
                wait();
                if (!ok) base = own = CUDART_NAN_F;
#pragma unroll 1
                for (int cb = 0; cb < 2; ++cb) {              // (128 columns at a time, half of them here)
                    const int c0 = t.n * kTileN + cb * 128, mine0 = c0 + half * 64;
                    uint32_t v[2][32], y[32];
                    tmem_columns32(tile_at() + cb * 128 + half * 64, v[0]);
                    tmem_columns32(tile_at() + cb * 128 + half * 64 + 32, v[1]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (cb == 1) taken();
                    if (rows <= 0) continue;
                    if (chunks > 1) { add_earlier(v[0], 2 * cb); add_earlier(v[1], 2 * cb + 1); }
                    const int at = target - mine0;
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        float f[2];
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            const int col = 2 * e + o;
                            const float s = exp2_fast(fmaf(__uint_as_float(v[col >> 5][col & 31]), p.c, -base));
                            f[o] = counts ? (at == col ? own : s) : 0.f;
                        }
                        const __nv_bfloat162 b = __floats2bfloat162_rn(f[0], f[1]);
                        y[e] = *reinterpret_cast<const uint32_t*>(&b);
                    }
                    // (behind the last column the contraction meets zeros, but not with an infinity: 0 there may lie far above a row's logits)
                    if (mine0 + 64 > of.N) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) y[e] &= mine0 + 2 * e + 1 < of.N ? 0xffffffffu : mine0 + 2 * e < of.N ? 0xffffu : 0u;
                    }
                    store_128(panel, y, p.p, p.ldp, row0, rows, c0, 128, true, q, half, lane);
                }
            } else if (!t.head) {
                const int rr = lane >> 3, ch = lane & 7;
                float* const acc = p.acc + (size_t)t.share * of.M * p.ld_acc;
#pragma unroll 1
                for (int c = 0; c < 4 * chunks; ++c) {        // (a longer contraction is added to what is there, as that of later pieces of the vocabulary)
                    const int cb = c & 3;
                    if (cb == 0) wait();
                    const int n = n0 + cb * 32 + 4 * ch;
                    uint32_t v[32];
                    tmem_columns32(from() + cb * 32, v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (cb == 3) taken();
                    if (n0 + cb * 32 >= p.ld_acc || rows <= 0) continue;
#pragma unroll
                    for (int g = 0; g < 8; ++g)
                        *reinterpret_cast<uint4*>(blk + lane * 128 + ((g ^ (lane & 7)) << 4)) = make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int r = 4 * e + rr;
                        if (r >= rows || n >= p.ld_acc) break;
                        float4 f = *reinterpret_cast<const float4*>(blk + r * 128 + ((ch ^ (r & 7)) << 4));
                        float4* const to = reinterpret_cast<float4*>(acc + (size_t)(row0 + r) * p.ld_acc + n);
                        if (!ok) f.x = f.y = f.z = f.w = CUDART_NAN_F;
                        if (p.add || c > 3) {
                            const float4 o = *to;
                            f.x += o.x; f.y += o.y; f.z += o.z; f.w += o.w;
                        }
                        *to = f;
                    }
                    __syncwarp();
                }
                panel_sync(q);                                // (the other warp's share is a panel's too)
            } else {
                earlier();
                wait();
                if (!ok) factor = CUDART_NAN_F;
#pragma unroll 1
                for (int cb = 0; cb < 2; ++cb) {
                    const int c0 = t.n * kTileN + cb * 128;
                    uint32_t v[2][32], y[32];
                    tmem_columns32(tile_at() + cb * 128 + half * 64, v[0]);
                    tmem_columns32(tile_at() + cb * 128 + half * 64 + 32, v[1]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (cb == 1) taken();
                    if (c0 >= of.N || rows <= 0) continue;
                    if (chunks > 1) { add_earlier(v[0], 2 * cb); add_earlier(v[1], 2 * cb + 1); }
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(v[e >> 4][2 * e & 31]) * factor, __uint_as_float(v[e >> 4][(2 * e & 31) + 1]) * factor);
                        y[e] = *reinterpret_cast<const uint32_t*>(&b);
                    }
                    store_128(panel, y, p.out, of.N, row0, rows, c0, of.N - c0, p.wide, q, half, lane);
                }
            }
        }
    }
    if (!ok && lane == 0) {
        if constexpr (PAIR) pair_gave_up(end);
        if (p.ran_out) {
            *reinterpret_cast<volatile int*>(p.ran_out) = 1;
            __threadfence_system();
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    // neither CTA's memory goes while the other still reads it or arrives there
    if constexpr (PAIR) pair_end(end, rank, full, kStages, kStage);
    else __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512));
    }
}

// Few rows (a token or some, up to 32): the head is the 128-row operand and streams once, the rows are the columns; float32 rows have a column for each of their three
// terms.  A CTA walks tiles of 128 head rows, and a thread keeps for its head row of every tile, per row of h, the largest logit and the sum of the exponentials below it;
// at the end the CTA's 128 threads meet.
//   warp 0    one lane: the head's tile [128 x 64] of a k-block and the rows' [columns x 64] into a ring
//   warp 1    MMAs (M = 128, N = the columns), an accumulator for 16 k-blocks
//   warps 2-5 take the accumulators out
// Bound: the head's bytes.  Tensor memory is taken behind the wait for the predecessor and in front of the signal to the successor (see the few rows of 4-bit numbers).
constexpr int kFewMost = 32, kFewCtas = 2 * 148, kFewThreads = 192, kFewCols = 256, kFewSlotsMost = 6, kFewChunk = 16;

template <int NB, int TERMS>
struct Few {
    static constexpr int kCols = NB * TERMS, kSlot = kTileBytes + kCols * 128, kFit = 110 * 1024 / kSlot, kSlots = kFit < kFewSlotsMost ? kFit : kFewSlotsMost;
    static constexpr int kSmem = kSlots * kSlot + 1024;
    static_assert(2 * kCols <= kFewCols && 2 * kFewCols <= 512 && 3 * kSmem > 228 * 1024, "two CTAs on an SM");
};

template <int NB, int TERMS>
__global__ void __launch_bounds__(kFewThreads, 2) loss_few_rows_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w,
                                                                       const __grid_constant__ LossTiles p) {
    constexpr int kCols = Few<NB, TERMS>::kCols, kSlot = Few<NB, TERMS>::kSlot, kSlots = Few<NB, TERMS>::kSlots;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[kSlots], empty[kSlots], t_full[2], t_empty[2], done;
    __shared__ uint32_t tmem_slot;
    __shared__ int targets[NB];
    __shared__ float2 meet[4][NB];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, M = p.own.M;
    const int n_kb = (p.own.K + kBK - 1) / kBK, n_tiles = (p.own.N + 127) / 128, mine = (n_tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x, blocks = mine * n_kb;
    const auto head_tile = [&](int slot, int t, int kb) {
        mbar_arrive_expect_tx(&full[slot], kSlot);
        tma_load_2d(smem_u32(smem + slot * kSlot), &map_w, smem_u32(&full[slot]), kb * kBK, t * 128);
    };
    const auto row_tile = [&](int slot, int kb) {
#pragma unroll
        for (int tm = 0; tm < TERMS; ++tm)
            tma_load_2d(smem_u32(smem + slot * kSlot + kTileBytes + tm * NB * 128), &map_h, smem_u32(&full[slot]), kb * kBK, tm * M);
    };
    int t = blockIdx.x, kb = 0;                               // of the next block that is asked for
    const auto next = [&]() {
        if (++kb == n_kb) kb = 0, t += gridDim.x;
    };
    if (tid == 0) {
        for (int i = 0; i < kSlots; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&t_full[i], 1); mbar_init(&t_empty[i], 4); }
        mbar_init(&done, 1);
        fence_mbar_init();
    }
    // (the head may be what the predecessor writes: a gradient, another product's result)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x == 0 && tid == 0) *p.arrived = 0u;
    if (tid == 0)
        for (int i = 0; i < min(blocks, kSlots); ++i) { head_tile(i, t, kb); row_tile(i, kb); next(); }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kFewCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    if (tid < NB) {
        const long long t = tid < M ? target_of(p.targets, p.targets64, tid) : -1;
        targets[tid] = t >= 0 && t < p.own.N ? (int)t : -1;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            int i = min(blocks, kSlots);
            for (; i < blocks; ++i) {
                const int slot = i % kSlots;
                if (!lane_wait(&empty[slot], ((i / kSlots) & 1u) ^ 1u, p.polls)) { ok = false; break; }
                head_tile(slot, t, kb);
                row_tile(slot, kb);
                next();
            }
            copies_landed(full, kSlots, i);
        }
    } else if (warp == 1) {
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kCols >> 3) << 17) | (8u << 24);
        unsigned it = 0;
        kb = 0;
        for (int i = 0; i < blocks && ok; ++i, kb = kb + 1 == n_kb ? 0 : kb + 1) {
            const int slot = i % kSlots;
            const bool first = kb % kFewChunk == 0, last = kb == n_kb - 1 || kb % kFewChunk == kFewChunk - 1;
            if (first) ok = pair_wait(&t_empty[it & 1u], ((it >> 1) & 1u) ^ 1u, p.polls);
            ok = ok && pair_wait(&full[slot], (i / kSlots) & 1u, p.polls);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = smem_u32(smem + slot * kSlot);
            const uint64_t adesc = umma_desc(at), bdesc = umma_desc(at + kTileBytes);
            if (elect_one_sync()) {
#pragma unroll
                for (int j = 0; j < kBK / 16; ++j) umma_bf16(tmem + (it & 1u) * kCols, adesc + 2 * j, bdesc + 2 * j, idesc, j != 0 || !first ? 1u : 0u);
                umma_commit(&empty[slot]);
                if (last) umma_commit(&t_full[it & 1u]);
            }
            __syncwarp();
            if (last) ++it;
        }
        mmas_ended<false>(&done);
    } else {
        const int q = warp & 3, c = q * 32 + lane;
        float most[NB], sum[NB];                              // of c z, of 2^(c z - most)
#pragma unroll
        for (int m = 0; m < NB; ++m) most[m] = -CUDART_INF_F, sum[m] = 0.f;
        unsigned it = 0;
        for (int j = 0; j < mine; ++j) {
            const int n = (blockIdx.x + j * gridDim.x) * 128 + c;
            float z[NB];
#pragma unroll
            for (int m = 0; m < NB; ++m) z[m] = 0.f;
            for (int kb = 0; kb < n_kb; kb += kFewChunk, ++it) {
                ok = ok && pair_wait(&t_full[it & 1u], (it >> 1) & 1u, p.polls);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int tm = TERMS - 1; tm >= 0; --tm)
#pragma unroll
                    for (int m0 = 0; m0 < NB; m0 += 16) {
                        uint32_t v[16];
                        tmem_columns16(tmem + ((uint32_t)(q * 32) << 16) + (it & 1u) * kCols + tm * NB + m0, v);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int e = 0; e < 16; ++e) z[m0 + e] += __uint_as_float(v[e]);
                    }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&t_empty[it & 1u]);
            }
            // (rows eight at a time, side by side: one after the other each took 0.2 us a tile and as much again at the end)
#pragma unroll
            for (int m0 = 0; m0 < NB; m0 += 8) {
                if (m0 >= M) break;
#pragma unroll
                for (int m = m0; m < m0 + 8; ++m) {
                    if (targets[m] == n) p.hit[m] = ok ? z[m] : CUDART_NAN_F;
                    const float now = fmaxf(most[m], n < p.own.N ? z[m] * p.c : -CUDART_INF_F), below = now == -CUDART_INF_F ? 0.f : now;
                    sum[m] = sum[m] * exp2_fast(most[m] - below) + exp2_fast(n < p.own.N ? fmaf(z[m], p.c, -below) : -CUDART_INF_F);
                    most[m] = now;
                }
            }
        }
#pragma unroll
        for (int m0 = 0; m0 < NB; m0 += 8) {
            if (m0 >= M) break;
            float top[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) top[m] = most[m0 + m];
#pragma unroll
            for (int o = 16; o; o >>= 1)
#pragma unroll
                for (int m = 0; m < 8; ++m) top[m] = fmaxf(top[m], __shfl_xor_sync(0xffffffffu, top[m], o));
#pragma unroll
            for (int m = 0; m < 8; ++m) sum[m0 + m] *= exp2_fast(most[m0 + m] - (top[m] == -CUDART_INF_F ? 0.f : top[m]));
#pragma unroll
            for (int o = 16; o; o >>= 1)
#pragma unroll
                for (int m = 0; m < 8; ++m) sum[m0 + m] += __shfl_xor_sync(0xffffffffu, sum[m0 + m], o);
            if (lane == 0) {
#pragma unroll
                for (int m = 0; m < 8; ++m) meet[q][m0 + m] = ok ? make_float2(top[m], sum[m0 + m]) : make_float2(CUDART_NAN_F, CUDART_NAN_F);
            }
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
    for (int i = tid; i < 4 * M; i += kFewThreads) p.part[((size_t)(i >> 2) * gridDim.x + blockIdx.x) * 4 + (i & 3)] = meet[i & 3][i >> 2];
}

// The tiles of a row joined, a warp per row; where their sum or mean is asked for, the last block to come sums the rows, in their order.
// (part, hit: their writer may still run when this kernel starts, so not by the read-only path, which __restrict__ would allow)
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(32 * kJoinWarps) loss_join_kernel(const float2* part, const float* hit, int M, int V, int tiles, const void* targets,
                                                                    int targets64, long long ignore, float c, int reduction, float* __restrict__ out, float2* kept,
                                                                    unsigned* arrived) {
    const int lane = threadIdx.x & 31, row = blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");        // (launched while the tiles are on their way)
    if (row < M) {
        const float2* const p = part + (size_t)row * tiles;
        float most = -CUDART_INF_F, sum = 0.f;
        bool bad = false;
        for (int i = lane; i < tiles; i += 32) {
            const float2 x = p[i];
            const float now = fmaxf(most, x.x);
            bad = bad || x.y != x.y || x.x != x.x;
            if (now > -CUDART_INF_F) sum = sum * exp2f(most - now) + x.y * exp2f(x.x - now);
            most = now;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, most, o), add = __shfl_xor_sync(0xffffffffu, sum, o), now = fmaxf(most, other);
            if (now > -CUDART_INF_F) sum = sum * exp2f(most - now) + add * exp2f(other - now);
            most = now;
        }
        bad = __any_sync(0xffffffffu, bad);
        if (lane == 0) {
            const long long t = target_of(targets, targets64, row);
            const float below = bad ? CUDART_NAN_F : log2f(sum);
            // (the target's distance from the largest is taken before it meets the logarithm: losses near zero keep their digits)
            const float l = t == ignore ? 0.f : t < 0 || t >= V ? CUDART_NAN_F : (below - fmaf(hit[row], c, -most)) * kLn2;
            kept[row] = make_float2((most + below) * kLn2, l);
            if (reduction == kLossEach) out[row] = l;
        }
    }
    if (reduction == kLossEach) return;
    __shared__ bool last;
    __shared__ int counts[kJoinWarps];
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(arrived, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    // every thread its rows in double precision, then a fixed tree
    double s = 0.0;
    int n = 0;
    for (int i = threadIdx.x; i < M; i += 32 * kJoinWarps)
        if (target_of(targets, targets64, i) != ignore) {
            s += (double)__ldcg(&kept[i].y);
            ++n;
        }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        n += __shfl_xor_sync(0xffffffffu, n, o);
    }
    __shared__ double parts[kJoinWarps];
    if (lane == 0) { parts[threadIdx.x >> 5] = s; counts[threadIdx.x >> 5] = n; }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        n = 0;
        for (int i = 0; i < kJoinWarps; ++i) { s += parts[i]; n += counts[i]; }
        *out = reduction == kLossSum ? (float)s : n ? (float)(s / n) : 0.f;
        *reinterpret_cast<float*>(kept + M) = (float)n;
    }
}

// Rows as operands: out [TERMS][M][ld_out] bf16, zeros from K on.  TERMS 3: fp32 rows as three bf16 terms (24 bits).  targets: rows whose target is `ignore` are zeros
// (what they hold, a NaN among it, stays out of the head's gradient).  grad: the others times grad scale [/ *count] of their own.
template <int TERMS, bool F32>
__global__ void __launch_bounds__(256) loss_pack_kernel(const void* __restrict__ x, long long ld, int M, int K, __nv_bfloat16* __restrict__ out, int ld_out, const void* targets,
                                                        int targets64, long long ignore, const float* grad, int grad_stride, const float* count, float scale) {
    const int per_row = ld_out / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, r = i / per_row;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (r >= M) return;
    const int k = (int)(i - r * per_row) * 8;
    const bool out_of_it = targets && target_of(targets, targets64, (int)r) == ignore;
    float factor = 1.f;
    if (grad) {
        factor = grad[r * grad_stride] * scale;
        if (count) factor /= fmaxf(*count, 1.f);
    }
    __nv_bfloat16 t[TERMS][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v = 0.f;
        if (k + e < K && !out_of_it) v = F32 ? reinterpret_cast<const float*>(x)[r * ld + k + e] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(x)[r * ld + k + e]);
        if (grad && !out_of_it) v *= factor;
        t[0][e] = TERMS == 1 ? __float2bfloat16_rn(v) : __float2bfloat16_rz(v);
        if (TERMS == 3) {                                     // rounded towards zero first: the largest numbers do not become infinities
            const float f = __bfloat162float(t[0][e]), r1 = fabsf(f) <= 3.402823466e38f ? v - f : 0.f;
            t[TERMS > 1][e] = __float2bfloat16_rn(r1);
            t[TERMS - 1][e] = __float2bfloat16_rn(r1 - __bfloat162float(t[TERMS > 1][e]));
        }
    }
#pragma unroll
    for (int q = 0; q < TERMS; ++q) *reinterpret_cast<uint4*>(out + ((size_t)q * M + r) * ld_out + k) = *reinterpret_cast<const uint4*>(t[q]);
}

// dh = the sum of the shares of the contraction, times grad scale [/ *count]  (acc, grad and count: as part and hit above)
__global__ void __launch_bounds__(256) loss_rows_out_kernel(const float* acc, int splits, int M, int K, int ld, __nv_bfloat16* __restrict__ out, int wide,
                                                            const float* grad, int grad_stride, const float* count, float scale, const void* targets,
                                                            int targets64, long long ignore) {
    const int per_row = ld / 4;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, r = i / per_row;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (r >= M) return;
    const int k = (int)(i - r * per_row) * 4;
    float4 v = *reinterpret_cast<const float4*>(acc + r * ld + k);
    for (int s = 1; s < splits; ++s) {
        const float4 o = *reinterpret_cast<const float4*>(acc + ((size_t)s * M + r) * ld + k);
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
    }
    float f = grad[r * grad_stride] * scale;
    if (count) f /= fmaxf(*count, 1.f);
    if (target_of(targets, targets64, (int)r) == ignore) f = 0.f;
    v.x *= f; v.y *= f; v.z *= f; v.w *= f;
    const __nv_bfloat16 h[4] = {__float2bfloat16_rn(v.x), __float2bfloat16_rn(v.y), __float2bfloat16_rn(v.z), __float2bfloat16_rn(v.w)};
    __nv_bfloat16* const o = out + (size_t)r * K + k;
    if (wide) {
        *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(h);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (k + e < K) o[e] = h[e];
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------------

// bf16 [rows][cols], ld elements apart, in boxes of box_rows x 64 columns
bool bf16_map(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld, int box_rows) {
    const EncodeTiledFn enc = encode_tiled();
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {kBK, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// a launch that may start while its predecessor still runs (every kernel here waits for it where it has to)
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), unsigned grid, unsigned threads, size_t smem, cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

template <int KIND, int TERMS>
cudaError_t pairs_of(int dev, int* out) {
    static std::atomic<int> known[64];
    if (dev >= 0 && dev < 64 && (*out = known[dev].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
    const auto kernel = loss_product_kernel<KIND, TERMS>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Ring<TERMS, true>::kSmem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<TERMS, true>::kSmem);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(out, kernel, &cfg);
    if (e != cudaSuccess) return e;
    if (*out < 1) return cudaErrorNotSupported;
    if (dev >= 0 && dev < 64) known[dev].store(*out, std::memory_order_relaxed);
    return cudaSuccess;
}

// (hs, ht: the operands of dw in kGrads).  128 rows and less of logits go on one SM per tile
template <int KIND, int TERMS>
cudaError_t run_tiles(const CUtensorMap& a, const CUtensorMap& b, LossTiles p, int dev, cudaStream_t st, const CUtensorMap* hs = nullptr, const CUtensorMap* ht = nullptr) {
    p.polls = gemm_pair_polls();
    p.ran_out = split_attention_ran_out(dev, st);
    p.own.rows = p.head.rows = 256;
    if constexpr (KIND != kGrads) {
        if (p.own.M <= 128) {
            int sms = 0;
            cudaError_t e = current_sms(&dev, &sms);
            if (e == cudaSuccess) e = ask_smem<loss_product_kernel<KIND, TERMS, false>>(dev, Ring<TERMS, false>::kSmem);
            if (e != cudaSuccess) return e;
            p.own.rows = 128;
            p.many = p.own.tiles_n();
            return launch_early(loss_product_kernel<KIND, TERMS, false>, std::min(p.many, p.sums ? std::min(sms, kSumsCtas) : sms), kThreads, Ring<TERMS, false>::kSmem, st, a, b, a, b, p);
        }
    }
    int pairs = 0;
    const cudaError_t e = pairs_of<KIND, TERMS>(dev, &pairs);
    if (e != cudaSuccess) return e;
    if (p.sums) pairs = std::min(pairs, kSumsCtas / 2);
    const long long own = p.own.tiles(), head = p.head.tiles();
    if (own + head > 0x3fffffffLL) return cudaErrorNotSupported;
    // what a tile takes, in k-blocks; taking it out lasts as long as eight of them
    const int long_own = std::max(p.own.share(), 8), long_head = std::max(p.head.blocks(), 8);
    p.first_head = own == 0 || (head > 0 && long_head > long_own);
    p.many = (int)(p.first_head ? head : own);
    p.extra = own && head ? std::max(1, (p.first_head ? long_head + long_own / 2 : long_own + long_head / 2) / (p.first_head ? long_own : long_head)) : 0;
    return launch_early(loss_product_kernel<KIND, TERMS>, 2 * (int)std::min<long long>(own + head, pairs), kThreads, Ring<TERMS, true>::kSmem, st, a, b, hs ? *hs : a, ht ? *ht : b, p);
}

template <int NB, int TERMS>
cudaError_t run_few(const CUtensorMap& h, const CUtensorMap& w, LossTiles p, int grid, int dev, cudaStream_t st) {
    const cudaError_t e = ask_smem<loss_few_rows_kernel<NB, TERMS>>(dev, Few<NB, TERMS>::kSmem);
    if (e != cudaSuccess) return e;
    p.polls = gemm_pair_polls();
    p.ran_out = split_attention_ran_out(dev, st);
    return launch_early(loss_few_rows_kernel<NB, TERMS>, grid, kFewThreads, Few<NB, TERMS>::kSmem, st, h, w, p);
}

int padded(int K) { return (K + 7) / 8 * 8; }
bool in_place(const void* x, long long ld) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld % 8 == 0; }
size_t up(size_t n) { return (n + 255) / 256 * 256; }

template <int TERMS, bool F32>
cudaError_t pack(const void* x, long long ld, int M, int K, void* out, const LossShape* counts, cudaStream_t st, const LossGrad* by = nullptr) {
    const long long blocks = ((long long)M * (padded(K) / 8) + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
    loss_pack_kernel<TERMS, F32><<<(unsigned)blocks, 256, 0, st>>>(x, ld, M, K, reinterpret_cast<__nv_bfloat16*>(out), padded(K), counts ? counts->targets : nullptr,
                                                                   counts ? counts->targets64 : 0, counts ? counts->ignore : 0, by ? by->grad : nullptr, by ? by->grad_stride : 0,
                                                                   by ? by->count : nullptr, counts ? counts->scale : 1.f);
    ++extra_launches();
    return cudaGetLastError();
}

// Shares of a contraction of `length`, none of them empty, where `most` are asked for
int shares_of(int length, int most) {
    const int kb = (length + kBK - 1) / kBK, per = (kb + most - 1) / most;
    return (kb + per - 1) / per;
}

// What a call keeps in its workspace, one after the other
struct Room {
    size_t h = 0, h_dw = 0, w = 0, part = 0, hit = 0, arrived = 0, kept = 0, p = 0, acc = 0, sums = 0, all = 0;      // offsets
    bool few = false, long_p = false, long_dw = false;                                  // (contractions that an accumulator does not take)
    int parts = 0;                                                                      // of a row's logits
    int piece = 0, splits = 1;                                                          // columns of a piece of the vocabulary, shares of dh's contraction
};
Room room_of(const LossShape& s, bool grad, bool rows, bool head) {
    Room r;
    size_t at = 0;
    const auto take = [&](size_t bytes) { const size_t was = at; at += up(bytes); return was; };
    const size_t row = (size_t)s.M * padded(s.K) * 2;
    r.h = take(s.h_type == kTypeF32 ? 3 * row : in_place(s.h, s.ldh) ? 0 : row);
    r.h_dw = take(grad && head ? row : 0);
    r.w = take(in_place(s.w, s.ldw) ? 0 : (size_t)s.V * padded(s.K) * 2);
    if (!grad) {
        r.few = s.M <= kFewMost;
        r.parts = r.few ? (int)std::min<long long>((s.V + 127LL) / 128, kFewCtas) * 4 : 2 * ((s.V + kTileN - 1) / kTileN);
        r.part = take((size_t)s.M * r.parts * 8);
        r.hit = take((size_t)s.M * 4);
        r.arrived = take(4);
        r.kept = take((size_t)s.M * 8 + 4);
    } else {
        const long long all = (s.V + 255) / 256 * 256LL, fit = (128LL << 20) / 2 / s.M / 256 * 256;
        r.piece = (int)std::min(all, std::max(4096LL, fit));
        // shares of dh's contraction where its tiles leave most of the chip idle
        const long long tiles = (long long)((s.M + 255) / 256) * ((s.K + 255) / 256);
        while (r.splits < 16 && 2 * r.splits * tiles <= 74 && r.piece / kBK >= 16 * r.splits) r.splits *= 2;
        // (of the columns that are there, not of the padded piece: the first piece writes every share, later ones add to the first of them)
        r.splits = shares_of(std::min(r.piece, s.V), r.splits);
        r.p = take((size_t)s.M * r.piece * 2);
        r.acc = take(rows ? (size_t)r.splits * s.M * ((s.K + 3) / 4 * 4) * 4 : 0);
        r.long_p = s.K > kChunkOf<kProbs, 1> * kBK;
        r.long_dw = head && s.M > kChunkOf<kGrads, 1> * kBK;
        r.sums = take(r.long_p || r.long_dw ? (size_t)kSumsCtas * kSumsFloats * 4 : 0);
    }
    r.all = at;
    return r;
}

LossTiles tiles_of(const LossShape& s) {
    LossTiles p{};
    p.own.splits = p.head.splits = 1;
    p.targets = s.targets; p.targets64 = s.targets64; p.ignore = s.ignore;
    p.c = s.scale * kLog2e; p.V = s.V;
    return p;
}

}  // namespace

bool loss_reads(const void* x, long long ld) { return in_place(x, ld); }
int loss_row(int K) { return padded(K); }
cudaError_t launch_loss_lay_out(const void* x, long long ld, int rows, int K, void* out, cudaStream_t st) {
    const cudaError_t e = pack<1, false>(x, ld, rows, K, out, nullptr, st);
    --extra_launches();                                       // (the caller counts one)
    return e;
}

size_t loss_work_bytes(const LossShape& s) { return room_of(s, false, false, false).all; }
size_t loss_grad_work_bytes(const LossShape& s, bool rows, bool head) { return room_of(s, true, rows, head).all; }

cudaError_t launch_loss(const LossShape& s, int reduction, float* out, float* kept, void* work, cudaStream_t st) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (take_ran_out(dev, st)) return cudaErrorLaunchTimeout;
    const Room r = room_of(s, false, false, false);
    unsigned char* const base = reinterpret_cast<unsigned char*>(work);
    const void *h = s.h, *w = s.w;
    long long ldh = s.ldh, ldw = s.ldw;
    const bool f32 = s.h_type == kTypeF32;
    if (f32 || !in_place(s.h, s.ldh)) {
        h = base + r.h;
        ldh = padded(s.K);
        e = f32 ? pack<3, true>(s.h, s.ldh, s.M, s.K, base + r.h, nullptr, st) : pack<1, false>(s.h, s.ldh, s.M, s.K, base + r.h, nullptr, st);
    }
    if (e == cudaSuccess && !in_place(s.w, s.ldw)) {
        w = base + r.w;
        ldw = padded(s.K);
        e = pack<1, false>(s.w, s.ldw, s.V, s.K, base + r.w, nullptr, st);
    }
    if (e != cudaSuccess) return e;
    const int columns = s.M <= 16 ? 16 : 32;
    CUtensorMap ma, mb;
    if (!bf16_map(&ma, h, (long long)s.M * (f32 ? 3 : 1), s.K, ldh, r.few ? columns : 128) || !bf16_map(&mb, w, s.V, s.K, ldw, 128)) return cudaErrorNotSupported;
    LossTiles p = tiles_of(s);
    p.own.M = s.M; p.own.N = s.V; p.own.K = s.K;
    p.part = reinterpret_cast<float2*>(base + r.part);
    p.hit = reinterpret_cast<float*>(base + r.hit);
    p.arrived = reinterpret_cast<unsigned*>(base + r.arrived);
    if (!r.few) e = f32 ? run_tiles<kStats, 3>(ma, mb, p, dev, st) : run_tiles<kStats, 1>(ma, mb, p, dev, st);
    else if (columns == 16) e = f32 ? run_few<16, 3>(ma, mb, p, r.parts / 4, dev, st) : run_few<16, 1>(ma, mb, p, r.parts / 4, dev, st);
    else e = f32 ? run_few<32, 3>(ma, mb, p, r.parts / 4, dev, st) : run_few<32, 1>(ma, mb, p, r.parts / 4, dev, st);
    if (e != cudaSuccess) return e;
    ++extra_launches();
    return launch_early(loss_join_kernel, (s.M + kJoinWarps - 1) / kJoinWarps, 32 * kJoinWarps, 0, st, p.part, p.hit, s.M, s.V, r.parts, s.targets, s.targets64, s.ignore, p.c,
                        reduction, out, kept ? reinterpret_cast<float2*>(kept) : reinterpret_cast<float2*>(base + r.kept), p.arrived);
}

cudaError_t launch_loss_grad(const LossShape& s, const float* kept, const LossGrad& by, void* dh, void* dw, void* work, cudaStream_t st) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (take_ran_out(dev, st)) return cudaErrorLaunchTimeout;
    const Room r = room_of(s, true, dh != nullptr, dw != nullptr);
    unsigned char* const base = reinterpret_cast<unsigned char*>(work);
    const void *h = s.h, *w = s.w;
    long long ldh = s.ldh, ldw = s.ldw;
    if (!in_place(s.h, s.ldh)) {
        h = base + r.h;
        ldh = padded(s.K);
        e = pack<1, false>(s.h, s.ldh, s.M, s.K, base + r.h, nullptr, st);
    }
    // the rows as dw takes them: those that do not count are zeros, factors of their own are in them
    if (e == cudaSuccess && dw) e = pack<1, false>(s.h, s.ldh, s.M, s.K, base + r.h_dw, &s, st, by.grad_stride ? &by : nullptr);
    if (e == cudaSuccess && !in_place(s.w, s.ldw)) {
        w = base + r.w;
        ldw = padded(s.K);
        e = pack<1, false>(s.w, s.ldw, s.V, s.K, base + r.w, nullptr, st);
    }
    if (e != cudaSuccess) return e;
    __nv_bfloat16* const probs = reinterpret_cast<__nv_bfloat16*>(base + r.p);
    float* const acc = reinterpret_cast<float*>(base + r.acc);
    const int ld_acc = (s.K + 3) / 4 * 4;
    CUtensorMap h_rows, w_rows, p_rows, h_cols, w_cols, p_cols;
    // rows along the contraction, and (the last two products) channels of a row in boxes of 64 x 64
    if (!bf16_map(&h_rows, h, s.M, s.K, ldh, 128) || !bf16_map(&w_rows, w, s.V, s.K, ldw, 128) || !bf16_map(&p_rows, probs, s.M, r.piece, r.piece, 128) ||
        (dw && !bf16_map(&h_cols, base + r.h_dw, s.M, s.K, padded(s.K), kBK)) || !bf16_map(&w_cols, w, s.V, s.K, ldw, kBK) || !bf16_map(&p_cols, probs, s.M, r.piece, r.piece, kBK))
        return cudaErrorNotSupported;
    for (long long from = 0; from < s.V; from += r.piece) {
        const int v0 = (int)from;
        const int cols = std::min(r.piece, s.V - v0);
        LossTiles p = tiles_of(s);
        p.v0 = v0;
        p.own.M = s.M; p.own.N = cols; p.own.K = s.K;
        p.kept = reinterpret_cast<const float2*>(kept);
        p.p = probs; p.ldp = r.piece;
        if (r.long_p) p.sums = reinterpret_cast<float*>(base + r.sums);
        e = run_tiles<kProbs, 1>(h_rows, w_rows, p, dev, st);
        if (e != cudaSuccess) return e;
        ++extra_launches();
        LossTiles q = tiles_of(s);
        q.v0 = v0;
        if (dh) {
            q.own.M = s.M; q.own.N = s.K; q.own.K = cols;
            q.own.splits = v0 ? shares_of(cols, r.splits) : r.splits;
            q.acc = acc; q.ld_acc = ld_acc; q.add = v0 > 0;
        }
        if (dw) {
            if (r.long_dw) q.sums = reinterpret_cast<float*>(base + r.sums);
            q.head.M = cols; q.head.N = s.K; q.head.K = s.M;
            q.out = reinterpret_cast<__nv_bfloat16*>(dw) + (size_t)v0 * s.K;
            if (!by.grad_stride) q.grad = by.grad, q.count = by.count, q.scale = s.scale;      // (else the rows have theirs)
            q.wide = s.K % 8 == 0 && (reinterpret_cast<uintptr_t>(dw) & 15) == 0;
        }
        e = run_tiles<kGrads, 1>(p_rows, w_cols, q, dev, st, &p_cols, dw ? &h_cols : nullptr);
        if (e != cudaSuccess) return e;
        ++extra_launches();
    }
    if (dh) {
        const long long blocks = ((long long)s.M * (ld_acc / 4) + 255) / 256;
        if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
        e = launch_early(loss_rows_out_kernel, (unsigned)blocks, 256, 0, st, acc, r.splits, s.M, s.K, ld_acc, reinterpret_cast<__nv_bfloat16*>(dh),
                         (int)(s.K % 4 == 0 && (reinterpret_cast<uintptr_t>(dh) & 7) == 0), by.grad, by.grad_stride, by.count, s.scale, s.targets, s.targets64, s.ignore);
        ++extra_launches();
    }
    --extra_launches();                                       // (the caller counts one)
    return e;
}

}  // namespace lm
