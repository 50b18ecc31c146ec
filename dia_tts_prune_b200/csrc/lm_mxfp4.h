// lm_mxfp4.h - rows in microscaled 4-bit numbers (MXFP4) and the product with a matrix of them.
//
// A row's channels go in blocks of 32 that share a power of two: value = e2m1 2^(scale - 127), scale 255 for a block that is not finite.
//   codes   [rows][stride / 2] bytes, two channels a byte, the lower one in the lower four bits; stride = channels padded to 128 with zeros
//   scales  [rows padded to 128 / 128][stride / 128][512] bytes: the scale of row r, block b of a piece of 128 rows x 128 channels stands at
//           (r % 32) 16 + (r / 32 % 4) 4 + b % 4, which is how a copy into tensor memory finds the rows of a tile
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace lm {

enum Mxfp4Type { kTypeF32 = 0, kTypeBf16 = 1, kTypeF16 = 2 };
inline int type_bytes(int type) { return type == kTypeF32 ? 4 : 2; }

constexpr int kMxStride = 128, kMxScaleBytes = 512;
inline long long mx_stride(long long K) { return (K + kMxStride - 1) / kMxStride * kMxStride; }
inline size_t mx_code_bytes(long long rows, long long K) { return (size_t)rows * (mx_stride(K) / 2); }
inline size_t mx_scale_bytes(long long rows, long long K) { return (size_t)((rows + 127) / 128) * (mx_stride(K) / kMxStride) * kMxScaleBytes; }

// x [rows][K], row stride ld elements.  early: a kernel launched behind it with programmatic serialization may start at once
cudaError_t launch_mxfp4_quantize(const void* x, int type, long long ld, int rows, int K, void* codes, void* scales, cudaStream_t st, bool early = false);
cudaError_t launch_mxfp4_dequantize(const void* codes, const void* scales, int rows, int K, void* out, int type, cudaStream_t st);

// Y[M][N] = Q(A)[M][K] W[N][K]^T with W in MXFP4, Q the rounding of A's rows to it, fp32 sums, Y in y_type (row stride N)
struct Mxfp4Product {
    const void* a; int a_type; long long lda;
    const void *w_codes, *w_scales;
    void* y; int y_type;
    int M, N, K;
    int* ran_out;
    unsigned polls;
};
size_t mxfp4_linear_work_bytes(int M, int N, int K);
cudaError_t launch_mxfp4_linear(Mxfp4Product p, void* work, cudaStream_t st);

}  // namespace lm
