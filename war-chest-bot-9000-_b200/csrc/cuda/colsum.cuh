// Column sums of a 32-bit matrix of partial results, in a fixed order.
#pragma once
#include "train.cuh"

namespace wctrain {

// out[k][c] = sum over s of part[s * ld + k * cols + c], k = blockIdx.y (an
// out that is null is not wanted): 32 columns a CTA, its rows dealt to
// blockDim.y warps and joined in order.
struct ColSums {
    float* out[4];
};
static __global__ void k_colsum(const float* __restrict__ part, int64_t splits, int64_t ld, int64_t cols, ColSums to) {
    __shared__ float s[32][33];
    float* out = to.out[blockIdx.y];
    if (!out) return;
    const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float v = 0.0f;
    if (c < cols)
        for (int64_t i = threadIdx.y; i < splits; i += blockDim.y) v += part[i * ld + blockIdx.y * cols + c];
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y == 0 && c < cols) {
        for (int j = 1; j < (int)blockDim.y; ++j) v += s[j][threadIdx.x];
        out[c] = v;
    }
}

inline void launch_colsum(const float* part, int64_t splits, int64_t ld, int64_t cols, int sums, const ColSums& to, cudaStream_t s) {
    if (!cols) return;
    const int rows = splits >= 16 ? 32 : 4;
    k_colsum<<<dim3((unsigned)((cols + 31) / 32), sums), dim3(32, rows), 0, s>>>(part, splits, ld, cols, to);
}

}  // namespace wctrain
