// lm_loss.h - cross entropy of rows under a head and its gradient, the logits in pieces that stay on the chip.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace lm {

// z[i][j] = scale h_i . w_j; loss_i = log sum_j exp z[i][j] - z[i][target_i], zero where the target is `ignore`
struct LossShape {
    const void* h; int h_type; long long ldh;    // [M][K] fp32 or bf16
    const void* w; long long ldw;                // [V][K] bf16
    const void* targets; int targets64;          // [M] int64 or int32
    long long ignore;
    int M, V, K;
    float scale;
};
// bf16 rows that the kernels read where they are: 16-byte aligned, a multiple of 8 elements apart.  Others are laid out again in the workspace of every call, or by the caller
// once for several, loss_row(K) elements apart with zeros behind the K-th
bool loss_reads(const void* x, long long ld);
int loss_row(int K);
cudaError_t launch_loss_lay_out(const void* x, long long ld, int rows, int K, void* out, cudaStream_t st);
size_t loss_work_bytes(const LossShape& s);
// out: every loss [M], or the sum or the mean (0 where none counts) of those that count.  kept [M][2] and one more (or null), for the gradient: log sum_j exp z[i][j] and the
// loss, and (not with kLossEach) how many rows count
enum LossReduction { kLossEach = 0, kLossSum = 1, kLossMean = 2 };
cudaError_t launch_loss(const LossShape& s, int reduction, float* out, float* kept, void* work, cudaStream_t st);

// The gradient by rows (dh [M][K] bf16) and by the head (dw [V][K] bf16), either or both; h is bf16
struct LossGrad {
    const float* grad; int grad_stride;          // of every loss, grad_stride floats apart (0: one for all)
    const float* count;                          // divides it where not null (kept + 2 M of a mean)
};
size_t loss_grad_work_bytes(const LossShape& s, bool rows, bool head);
cudaError_t launch_loss_grad(const LossShape& s, const float* kept, const LossGrad& by, void* dh, void* dw, void* work, cudaStream_t st);

}  // namespace lm
