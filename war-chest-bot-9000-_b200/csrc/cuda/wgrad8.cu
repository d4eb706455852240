// dw = x8^T dy with x8 kept in 8 bits, and db = the column sums of dy.
//
// A CTA owns a 64 x 64 tile of dw and a range of rows; the ranges' partial
// results are joined by a second kernel in a fixed order.
#include "colsum.cuh"

namespace wctrain {

namespace {

constexpr int TILE = 64, DEEP = 16, THREADS = 256;

template <class T>
__global__ void __launch_bounds__(THREADS) k_wgrad8(wc_act8_wgrad_args a, int64_t chunk_rows, float* part) {
    __shared__ float sx[DEEP][TILE], sy[DEEP][TILE];
    const int64_t k0 = (int64_t)blockIdx.x * TILE, n0 = (int64_t)blockIdx.y * TILE;
    const int64_t blocks = (a.k + 31) / 32, first = blockIdx.z * chunk_rows, last = min(first + chunk_rows, a.rows);
    const int tk = threadIdx.x / 16 * 4, tn = threadIdx.x % 16 * 4;
    float acc[4][4] = {}, db[4] = {};
    for (int64_t t0 = first; t0 < last; t0 += DEEP) {
        for (int i = threadIdx.x; i < DEEP * TILE; i += THREADS) {
            const int64_t t = t0 + i / TILE, k = k0 + i % TILE, n = n0 + i % TILE;
            float x = 0.0f, y = 0.0f;
            if (t < last && k < a.k) x = (float)a.q[t * blocks * 32 + k] * act8_unit(a.scale[t * blocks + k / 32]);
            if (t < last && n < a.n) y = to_f(static_cast<const T*>(a.dy)[t * a.ld_dy + n]);
            sx[i / TILE][i % TILE] = x, sy[i / TILE][i % TILE] = y;
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y = sy[d][tn + j];
                db[j] += y;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i][j] += sx[d][tk + i] * y;
            }
        __syncthreads();
    }
    float* to = part + (int64_t)blockIdx.z * (a.k + 1) * a.n;
    for (int j = 0; j < 4; ++j) {
        if (n0 + tn + j >= a.n) continue;
        for (int i = 0; i < 4; ++i)
            if (k0 + tk + i < a.k) to[(k0 + tk + i) * a.n + n0 + tn + j] = acc[i][j];
        if (blockIdx.x == 0 && tk == 0) to[a.k * a.n + n0 + tn + j] = db[j];
    }
}

int64_t tiles(int64_t n) { return (n + TILE - 1) / TILE; }
int64_t splits_of(const wc_act8_wgrad_args& a) {
    const int64_t t = tiles(a.k) * tiles(a.n), want = t >= 592 ? 1 : 592 / t, most = (a.rows + 255) / 256;
    return most < 1 ? 1 : most < want ? most : want;
}

template <class T>
void launch_type(const wc_act8_wgrad_args& a, cudaStream_t s) {
    const int64_t z = splits_of(a);
    float* part = static_cast<float*>(a.workspace);
    k_wgrad8<T><<<dim3((unsigned)tiles(a.k), (unsigned)tiles(a.n), (unsigned)z), THREADS, 0, s>>>(a, (a.rows + z - 1) / z, part);
    const int64_t ld = (a.k + 1) * a.n;
    if (a.out_type == WC_F32) launch_colsum<float>(part, z, ld, a.k * a.n, static_cast<float*>(a.dw), s);
    else if (a.out_type == WC_F16) launch_colsum<__half>(part, z, ld, a.k * a.n, static_cast<__half*>(a.dw), s);
    else launch_colsum<__nv_bfloat16>(part, z, ld, a.k * a.n, static_cast<__nv_bfloat16*>(a.dw), s);
    if (a.db) launch_colsum<float>(part + a.k * a.n, z, ld, a.n, a.db, s);
}

}  // namespace

uint64_t wgrad8_workspace(const wc_act8_wgrad_args& a) {
    return a.k && a.n ? (uint64_t)splits_of(a) * (a.k + 1) * a.n * sizeof(float) : 0;
}

void launch_wgrad8(const wc_act8_wgrad_args& a, cudaStream_t s) {
    if (a.type == WC_F32) launch_type<float>(a, s);
    else if (a.type == WC_F16) launch_type<__half>(a, s);
    else launch_type<__nv_bfloat16>(a, s);
}

}  // namespace wctrain
