// lm_kv8.h - keys and values of sequences in pages, 8 bits a number, and the attention that reads them.
//
//   keys, values  [pages][kv_heads][page_size][stride] codes (E4M3, or two's complement), stride = dim padded to 16 with zeros
//   scales        [pages][kv_heads] fp32, a power of two for the tokens of a page and head: value = code * scale.  NaN: the page's head stands for NaNs
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "lm_mxfp4.h"

namespace lm {

enum Kv8Format { kKvE4m3 = 0, kKvInt8 = 1 };
constexpr int kKvBlock = 16;                              // tokens that a kernel takes at a time: pages hold a multiple of them
constexpr int kKvMostDim = 256, kKvMostPage = 128, kKvMostHeads = 4096;

struct Kv8Cache {
    uint8_t *keys, *values;
    float *key_scales, *value_scales;
    int pages, kv_heads, page_shift, dim, stride, format;  // page_size = 1 << page_shift
};

// The rows of a step.  Sequence i has the rows first[i] .. first[i + 1] of the packed ones (first NULL: row i alone), at positions past[i] and on.  A token whose
// place lies beyond the table, or whose page is none of the pool's, is not there: it is not written, not seen, and reads as zeros; a sequence whose past is negative
// has no tokens.
struct Kv8Step {
    const int *table;                                     // [sequences][max_pages], table_ld apart
    long long table_ld;
    int max_pages;
    const int *past, *first;
    int sequences, rows;

#ifdef __CUDACC__
    __device__ __forceinline__ int begin(int i) const { return first ? min(max(first[i], 0), rows) : min(i, rows); }
    __device__ __forceinline__ int end(int i) const { return first ? min(max(first[i + 1], 0), rows) : min(i + 1, rows); }
    __device__ __forceinline__ int page(int i, long long slot, int pages) const {
        if (slot < 0 || slot >= max_pages) return -1;
        const int p = table[i * table_ld + slot];
        return (unsigned)p < (unsigned)pages ? p : -1;
    }
    // the sequence of a row, or -1
    __device__ __forceinline__ int sequence_of(int row) const {
        if (!first) return row < sequences ? row : -1;
        int lo = 0, hi = sequences;                       // first[lo] <= row < first[hi], if any
        if (row < first[0] || row >= first[sequences]) return -1;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= row) lo = mid;
            else hi = mid;
        }
        return lo;
    }
#endif
};

// rows [rows][kv_heads][dim] with neighbouring channels
struct Kv8Rows {
    const void* x;
    long long row, head;                                  // elements from one to the next
};

cudaError_t launch_kv8_append(const Kv8Cache& c, const Kv8Step& s, Kv8Rows k, Kv8Rows v, int type, cudaStream_t st);
// k, v [rows][kv_heads][dim] of `type`; past: the position of a sequence's first row
cudaError_t launch_kv8_read(const Kv8Cache& c, const Kv8Step& s, void* k, void* v, int type, cudaStream_t st);

struct Kv8Attention {
    Kv8Rows q;                                            // [rows][heads][dim]
    void* out;                                            // the same, packed
    int heads, type;
    float scale;
    int window;                                           // a row sees itself and window - 1 tokens in front; 0: all
    const float* sinks;                                   // [heads] one more logit in the denominator; NULL: none
    int few_most;                                         // (token, query head) pairs per key head of a sequence that tiles of 16 of them take; others go 256 at a time
    int whole;                                            // CTAs of a cluster that takes whole tiles; 0: tiles are shared
};
// (tokens: what a row of the table has room for; 0 bytes: none are needed)
size_t kv8_attention_work_bytes(int kv_heads, int dim, int rows, int heads, int type, int sequences, long long tokens);
cudaError_t launch_kv8_attention(const Kv8Cache& c, const Kv8Step& s, Kv8Attention a, void* work, cudaStream_t st);      // (sets few_most and whole)

// lm_kv8_tiles.cu: the sequences of more than few_most pairs; bf16 or fp16 rows, dim up to 128.  alone: nothing else zeroes the rows of no sequence
bool kv8_tiles_ok(int dim, int type);
size_t kv8_tiles_work_bytes(int dim);
constexpr int kKvTileCounters = 2 * 148;                  // zeros, two for every chunk of keys that an item may go in
cudaError_t launch_kv8_tiles(const Kv8Cache& c, const Kv8Step& s, const Kv8Attention& a, bool alone, void* work, unsigned* arrived, cudaStream_t st);

}  // namespace lm
