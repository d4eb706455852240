// Activations in 8 bits: blocks of 32 values along a row share a power-of-two
// unit (train.cuh act8_code), so a stored value is a whole number times that
// unit and is exact in bf16.
//
// All of these are bound by the bytes they move. A thread holds 8 consecutive
// values (16 bytes of a 16-bit type in one load, 8 bytes of q in one store)
// and 4 threads a block: the largest magnitude takes two shuffles. Magnitudes
// are compared as integers, where NaN is above infinity above the rest, so
// either shows in the block's code.
#include "colsum.cuh"

namespace wctrain {

namespace {

constexpr int THREADS = 256;

// 8 values of a row from column c on; past the width they are 0
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int64_t c, int64_t width, float* v) {
    if (VEC && c + 8 <= width) {
        alignas(16) T e[8];
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(p + c);
        } else {
            *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(p + c);
            *reinterpret_cast<uint4*>(e + 4) = *reinterpret_cast<const uint4*>(p + c + 4);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < width ? to_f(p[c + i]) : 0.0f;
    }
}
template <class T, bool VEC>
__device__ __forceinline__ void store8(T* p, int64_t c, int64_t width, const float* v) {
    if (VEC && c + 8 <= width) {
        alignas(16) T e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f<T>(v[i]);
        *reinterpret_cast<uint4*>(p + c) = *reinterpret_cast<const uint4*>(e);
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(p + c + 4) = *reinterpret_cast<const uint4*>(e + 4);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < width) p[c + i] = from_f<T>(v[i]);
    }
}

__device__ __forceinline__ void dequantise8(uint2 q, uint32_t code, float* v) {
    const float unit = act8_unit(code);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)(int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3))) * unit;
}

enum { PACK, UNPACK, GELU };

template <class T, bool VEC, int WHAT>
__global__ void __launch_bounds__(THREADS) k_act8(wc_act8_args a, uint32_t chunks, uint32_t total) {
    const uint32_t i = blockIdx.x * THREADS + threadIdx.x;
    const bool in = i < total;  // total is a multiple of 4: a block's threads are in or out together
    const uint32_t row = in ? i / chunks : 0, chunk = in ? i - row * chunks : 0;
    const int64_t c = (int64_t)chunk * 8;
    float v[8];
    if constexpr (WHAT == UNPACK) {
        if (!in) return;
        dequantise8(reinterpret_cast<const uint2*>(a.q)[i], a.scale[i >> 2], v);
        store8<T, VEC>(static_cast<T*>(a.out) + row * a.ld_out, c, a.width, v);
    } else {
        if (in) load8<T, VEC>(static_cast<const T*>(a.x) + row * a.ld_x, c, a.width, v);
        else
            for (float& x : v) x = 0.0f;
        if constexpr (WHAT == GELU) {
            if (a.bias && in)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (c + k < a.width) v[k] += a.bias[c + k];
            if (in) {
                float y[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = gelu(v[k]);
                store8<T, VEC>(static_cast<T*>(a.out) + row * a.ld_out, c, a.width, y);
            }
        }
        uint32_t code;
        const uint2 q = quantise8(v, &code);
        if (in) {
            reinterpret_cast<uint2*>(a.q)[i] = q;
            if ((i & 3) == 0) a.scale[i >> 2] = (uint8_t)code;
        }
    }
}

// dz = da GELU'(z8). The CTA's threads keep their columns and walk down the
// rows [blockIdx.y * chunk_rows, ...): `lanes` threads a row, each 8 columns.
template <class T, bool VEC>
__global__ void __launch_bounds__(THREADS) k_gelu8_backward(wc_act8_args a, int chunks, int lanes, int64_t chunk_rows,
                                                            float* part) {
    __shared__ float s[THREADS][9];
    const int per = THREADS / lanes, r = threadIdx.x / lanes, at = blockIdx.x * lanes + threadIdx.x % lanes;
    const bool in = r < per && at < chunks;
    const int64_t c = (int64_t)at * 8, first = blockIdx.y * chunk_rows, last = min(first + chunk_rows, a.rows);
    float acc[8] = {};
    if (in)
        for (int64_t t = first + r; t < last; t += per) {
            float d[8], z[8];
            load8<T, VEC>(static_cast<const T*>(a.x) + t * a.ld_x, c, a.width, d);
            dequantise8(reinterpret_cast<const uint2*>(a.q)[t * chunks + at], a.scale[(t * chunks + at) >> 2], z);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                d[k] *= gelu_slope(z[k]);
                acc[k] += d[k];
            }
            store8<T, VEC>(static_cast<T*>(a.out) + t * a.ld_out, c, a.width, d);
        }
    if (!part) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) s[threadIdx.x][k] = acc[k];
    __syncthreads();
    if (in && r == 0)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float v = acc[k];
            for (int j = 1; j < per; ++j) v += s[threadIdx.x + j * lanes][k];
            if (c + k < a.width) part[blockIdx.y * a.width + c + k] = v;
        }
}

bool aligned(const void* p, int64_t ld, size_t e) { return ((uintptr_t)p & 15) == 0 && (ld * e) % 16 == 0; }

template <int WHAT, class T>
void launch_as(const wc_act8_args& a, cudaStream_t s) {
    const int64_t chunks = (a.width + 31) / 32 * 4;
    // row and chunk come from one 32-bit index: longer calls go in ranges of rows
    const int64_t most = (1ll << 31) / chunks;
    for (int64_t t = 0; t < a.rows; t += most) {
        wc_act8_args b = a;
        b.rows = a.rows - t < most ? a.rows - t : most;
        if (a.x) b.x = static_cast<const T*>(a.x) + t * a.ld_x;
        if (a.out) b.out = static_cast<T*>(a.out) + t * a.ld_out;
        b.q += t * chunks * 8, b.scale += t * chunks / 4;
        const uint32_t total = (uint32_t)(b.rows * chunks), n = (total + THREADS - 1) / THREADS;
        const bool vec = (WHAT == UNPACK || aligned(b.x, a.ld_x, sizeof(T))) &&
                         (WHAT == PACK || aligned(b.out, a.ld_out, sizeof(T)));
        if (vec) k_act8<T, true, WHAT><<<n, THREADS, 0, s>>>(b, (uint32_t)chunks, total);
        else k_act8<T, false, WHAT><<<n, THREADS, 0, s>>>(b, (uint32_t)chunks, total);
    }
}
template <int WHAT>
void launch_type(const wc_act8_args& a, cudaStream_t s) {
    if (a.type == WC_F32) launch_as<WHAT, float>(a, s);
    else if (a.type == WC_F16) launch_as<WHAT, __half>(a, s);
    else launch_as<WHAT, __nv_bfloat16>(a, s);
}

struct Shape {
    int chunks, tiles, lanes, splits;
    int64_t chunk_rows;
    Shape(int64_t rows, int64_t width) {
        chunks = (int)((width + 31) / 32 * 4);
        tiles = (chunks + THREADS - 1) / THREADS;
        lanes = (chunks + tiles - 1) / tiles;
        const int per = THREADS / lanes;
        const int64_t want = (148 * 8 + tiles - 1) / tiles, most = (rows + 2 * per - 1) / (2 * per);
        splits = (int)(most < 1 ? 1 : most < want ? most : want);
        chunk_rows = (rows + splits - 1) / splits;
    }
};

template <class T>
void launch_backward(const wc_act8_args& a, cudaStream_t s) {
    const Shape g(a.rows, a.width);
    float* part = a.dbias ? static_cast<float*>(a.workspace) : nullptr;
    const bool vec = aligned(a.x, a.ld_x, sizeof(T)) && aligned(a.out, a.ld_out, sizeof(T));
    const dim3 grid(g.tiles, g.splits);
    if (vec) k_gelu8_backward<T, true><<<grid, THREADS, 0, s>>>(a, g.chunks, g.lanes, g.chunk_rows, part);
    else k_gelu8_backward<T, false><<<grid, THREADS, 0, s>>>(a, g.chunks, g.lanes, g.chunk_rows, part);
    if (part) launch_colsum<float>(part, g.splits, a.width, a.width, a.dbias, s);
}

}  // namespace

void launch_act8_pack(const wc_act8_args& a, cudaStream_t s) { launch_type<PACK>(a, s); }
void launch_act8_unpack(const wc_act8_args& a, cudaStream_t s) { launch_type<UNPACK>(a, s); }
void launch_gelu8(const wc_act8_args& a, cudaStream_t s) { launch_type<GELU>(a, s); }
uint64_t gelu8_workspace(int64_t rows, int64_t width) {
    return width ? (uint64_t)Shape(rows, width).splits * width * sizeof(float) : 0;
}
void launch_gelu8_backward(const wc_act8_args& a, cudaStream_t s) {
    if (a.type == WC_F32) launch_backward<float>(a, s);
    else if (a.type == WC_F16) launch_backward<__half>(a, s);
    else launch_backward<__nv_bfloat16>(a, s);
}

}  // namespace wctrain
