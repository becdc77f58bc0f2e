// Sums that several device operators end with.
#include "operators.h"

namespace {

// Partial matrices are as tall as a launch has blocks (some hundreds) and as wide as a model has parameters: a block takes 16
// neighbouring columns and reads 64 rows at a time, so that a column waits for memory a few times, not once per row (1170 x 640:
// 145 us with four rows at a time).  Joined in a fixed order.
constexpr int SUM_COLS = 16, SUM_ROWS = 64;
__global__ __launch_bounds__(1024) void sum_partials_kernel(const float* __restrict__ part, int64_t n_rows, int64_t n_cols, float* out0, int64_t n0,
                                                            float* out1, int64_t n1, float* out2)
{
    __shared__ double red[SUM_ROWS][SUM_COLS + 1];
    const int c = threadIdx.x % SUM_COLS, q = threadIdx.x / SUM_COLS;
    const int64_t col = (int64_t)blockIdx.x * SUM_COLS + c;
    double s = 0.0;
    if (col < n_cols) {
#pragma unroll 4
        for (int64_t r = q; r < n_rows; r += SUM_ROWS) s += part[r * n_cols + col];
    }
    red[q][c] = s;
    __syncthreads();
    for (int n = SUM_ROWS / 2; n > 0; n >>= 1) {
        if (q < n) red[q][c] += red[q + n][c];
        __syncthreads();
    }
    if (q != 0 || col >= n_cols) return;
    const float v = (float)red[0][c];
    if (col < n0) { if (out0) out0[col] = v; }
    else if (col < n0 + n1) { if (out1) out1[col - n0] = v; }
    else if (out2) out2[col - n0 - n1] = v;
}

}  // namespace

int64_t sum_partials_blocks(int64_t n_cols) { return (n_cols + SUM_COLS - 1) / SUM_COLS * (SUM_COLS * SUM_ROWS / 256); }

int launch_sum_partials(const float* part, int64_t n_rows, int64_t n_cols, float* out0, int64_t n0, float* out1, int64_t n1, float* out2, hipStream_t st)
{
    sum_partials_kernel<<<(unsigned)((n_cols + SUM_COLS - 1) / SUM_COLS), SUM_COLS * SUM_ROWS, 0, st>>>(part, n_rows, n_cols, out0, n0, out1, n1, out2);
    HIP_TRY(hipGetLastError());
    return 0;
}
