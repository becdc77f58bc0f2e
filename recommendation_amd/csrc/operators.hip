// Sums that several device operators end with.
#include "operators.h"

namespace {

// Partial matrices are as tall as a launch has blocks and as wide as a model has parameters: 64 neighbouring columns per
// block, its four wavefronts a quarter of the rows each, joined in a fixed order.
__global__ __launch_bounds__(256) void sum_partials_kernel(const float* __restrict__ part, int64_t n_rows, int64_t n_cols, float* out0, int64_t n0,
                                                           float* out1, int64_t n1, float* out2)
{
    __shared__ double red[4][64];
    const int64_t col = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const int q = threadIdx.x >> 6;
    double s = 0.0;
    if (col < n_cols)
        for (int64_t r = q; r < n_rows; r += 4) s += part[r * n_cols + col];
    red[q][threadIdx.x & 63] = s;
    __syncthreads();
    if (q != 0 || col >= n_cols) return;
    const int l = threadIdx.x;
    const float v = (float)((red[0][l] + red[1][l]) + (red[2][l] + red[3][l]));
    if (col < n0) { if (out0) out0[col] = v; }
    else if (col < n0 + n1) { if (out1) out1[col - n0] = v; }
    else if (out2) out2[col - n0 - n1] = v;
}

}  // namespace

int launch_sum_partials(const float* part, int64_t n_rows, int64_t n_cols, float* out0, int64_t n0, float* out1, int64_t n1, float* out2, hipStream_t st)
{
    sum_partials_kernel<<<(unsigned)((n_cols + 63) / 64), 256, 0, st>>>(part, n_rows, n_cols, out0, n0, out1, n1, out2);
    HIP_TRY(hipGetLastError());
    return 0;
}
