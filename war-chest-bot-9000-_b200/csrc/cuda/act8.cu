// Activations in 8 bits: blocks of 32 values along a row share a power-of-two
// unit (train.cuh act8_code), so a stored value is a whole number times that
// unit and is exact in bf16.
//
// All of these are bound by the bytes they move. Where addresses and strides
// allow, a thread holds 8 consecutive values (16 bytes of a 16-bit type in one
// load, 8 bytes of q in one store) and 4 threads a block: the largest magnitude
// takes two shuffles. Elsewhere a warp holds a block, one value a thread, so
// that its loads and stores are still next to each other.
#include <algorithm>

#include "colsum.cuh"

namespace wctrain {

namespace {

constexpr int THREADS = 256;

// 8 values of a row from column c on; those past the width (a whole number of 8s) are 0
template <class T>
__device__ __forceinline__ void load8(const T* p, int64_t c, int64_t width, float* v) {
    alignas(16) T e[8];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        reinterpret_cast<uint4*>(e)[i] = c < width ? __ldcs(reinterpret_cast<const uint4*>(p + c) + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f(e[i]);
}
template <class T>
__device__ __forceinline__ void store8(T* p, int64_t c, int64_t width, const float* v) {
    if (c >= width) return;
    alignas(16) T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f<T>(v[i]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) __stcs(reinterpret_cast<uint4*>(p + c) + i, reinterpret_cast<const uint4*>(e)[i]);
}

__device__ __forceinline__ void dequantise8(uint2 q, uint32_t code, float* v) {
    const float unit = act8_unit(code);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)(int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3))) * unit;
}

enum { PACK, UNPACK, GELU };

template <class T, int WHAT>
__global__ void __launch_bounds__(THREADS) k_act8(wc_act8_args a, uint32_t chunks, uint32_t total) {
    const uint32_t i = blockIdx.x * THREADS + threadIdx.x;
    const bool in = i < total;  // total is a multiple of 4: a block's threads are in or out together
    const uint32_t row = in ? i / chunks : 0, chunk = in ? i - row * chunks : 0;
    const int64_t c = (int64_t)chunk * 8;
    float v[8];
    if constexpr (WHAT == UNPACK) {
        if (!in) return;
        dequantise8(reinterpret_cast<const uint2*>(a.q)[i], a.scale[i >> 2], v);
        store8(static_cast<T*>(a.out) + row * a.ld_out, c, a.width, v);
    } else {
        load8(static_cast<const T*>(a.x) + row * a.ld_x, in ? c : a.width, a.width, v);
        if constexpr (WHAT == GELU) {
            if (in && c < a.width) {
                if (a.bias)
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] += a.bias[c + k];
                float y[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = gelu(v[k]);
                store8(static_cast<T*>(a.out) + row * a.ld_out, c, a.width, y);
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

// The same, a warp a run of 4 blocks of a row.
template <class T, int WHAT>
__global__ void __launch_bounds__(THREADS) k_act8_runs(wc_act8_args a, uint32_t blocks, uint32_t runs, uint32_t total) {
    const uint32_t i = (blockIdx.x * THREADS + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    if (i >= total) return;
    const int64_t row = i / runs;
    const uint32_t first = (i - (uint32_t)row * runs) * 4;
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t c = (int64_t)(first + k) * 32 + lane;
        v[k] = 0.0f;
        if (WHAT != UNPACK && c < a.width) v[k] = to_f(static_cast<const T*>(a.x)[row * a.ld_x + c]);
        if (WHAT == UNPACK && first + k < blocks) {
            const int64_t b = row * blocks + first + k;
            v[k] = (float)a.q[b * 32 + lane] * act8_unit(a.scale[b]);
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t c = (int64_t)(first + k) * 32 + lane, b = row * blocks + first + k;
        if (first + k >= blocks) break;
        if (WHAT == UNPACK) {
            if (c < a.width) static_cast<T*>(a.out)[row * a.ld_out + c] = from_f<T>(v[k]);
            continue;
        }
        if (WHAT == GELU && c < a.width) {
            if (a.bias) v[k] += a.bias[c];
            static_cast<T*>(a.out)[row * a.ld_out + c] = from_f<T>(gelu(v[k]));
        }
        const uint32_t code = act8_code(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v[k]) & 0x7fffffffu)));
        a.q[b * 32 + lane] = act8_whole(v[k], code);
        if (lane == 0) a.scale[b] = (uint8_t)code;
    }
}

// dz = da GELU'(z8). The CTA's threads keep their columns and walk down the
// rows [blockIdx.y * chunk_rows, ...): `lanes` threads a row, each 8 columns.
// UNITS: consecutive ones. Else `lanes` is a number of warps times 32, and a
// warp has 256 columns, thread by thread next to each other.
template <class T, bool UNITS>
__global__ void __launch_bounds__(THREADS) k_gelu8_backward(wc_act8_args a, int blocks, int lanes, int64_t chunk_rows, float* part) {
    __shared__ float s[THREADS][9];
    const int per = THREADS / lanes, r = threadIdx.x / lanes, at = blockIdx.x * lanes + threadIdx.x % lanes;
    const int step = UNITS ? 1 : 32, c = UNITS ? at * 8 : (at & ~31) * 8 + (at & 31);
    const bool in = r < per && c < a.width;
    const int64_t first = blockIdx.y * chunk_rows, last = min(first + chunk_rows, a.rows);
    float acc[8] = {};
    if (in)
        for (int64_t t = first + r; t < last; t += per) {
            const T* x = static_cast<const T*>(a.x) + t * a.ld_x;
            T* out = static_cast<T*>(a.out) + t * a.ld_out;
            float d[8], z[8];
            if constexpr (UNITS) {
                load8(x, c, a.width, d);
                dequantise8(*reinterpret_cast<const uint2*>(a.q + t * blocks * 32 + c), a.scale[t * blocks + c / 32], z);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const bool here = c + k * 32 < a.width;
                    d[k] = here ? to_f(x[c + k * 32]) : 0.0f;
                    z[k] = here ? (float)a.q[t * blocks * 32 + c + k * 32] * act8_unit(a.scale[t * blocks + c / 32 + k]) : 0.0f;
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                d[k] *= gelu_slope(z[k]);
                acc[k] += d[k];
            }
            if constexpr (UNITS) {
                store8(out, c, a.width, d);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (c + k * 32 < a.width) out[c + k * 32] = from_f<T>(d[k]);
            }
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
            if (c + k * step < a.width) part[blockIdx.y * a.width + c + k * step] = v;
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
        const bool units = a.width % 8 == 0 && (WHAT == UNPACK || aligned(b.x, a.ld_x, sizeof(T))) &&
                           (WHAT == PACK || aligned(b.out, a.ld_out, sizeof(T)));
        if (units) {
            const uint32_t total = (uint32_t)(b.rows * chunks);
            k_act8<T, WHAT><<<(total + THREADS - 1) / THREADS, THREADS, 0, s>>>(b, (uint32_t)chunks, total);
        } else {
            const uint32_t runs = (uint32_t)(chunks + 15) / 16, total = (uint32_t)(b.rows * runs);
            k_act8_runs<T, WHAT><<<(unsigned)((total + 7ull) / 8), THREADS, 0, s>>>(b, (uint32_t)(chunks / 4), runs, total);
        }
    }
}
template <int WHAT>
void launch_type(const wc_act8_args& a, cudaStream_t s) {
    if (a.type == WC_F32) launch_as<WHAT, float>(a, s);
    else if (a.type == WC_F16) launch_as<WHAT, __half>(a, s);
    else launch_as<WHAT, __nv_bfloat16>(a, s);
}

struct Shape {
    int blocks, tiles, lanes, splits;
    int64_t chunk_rows;
    Shape(int64_t rows, int64_t width, bool units) {
        blocks = (int)((width + 31) / 32);
        const int threads = units ? (int)(width / 8) : (int)((width + 255) / 256 * 32), whole = units ? 1 : 32;
        tiles = (threads + THREADS - 1) / THREADS;
        lanes = (threads / whole + tiles - 1) / tiles * whole;
        const int per = THREADS / lanes;
        const int64_t want = (148 * 8 + tiles - 1) / tiles, most = (rows + 2 * per - 1) / (2 * per);
        splits = (int)(most < 1 ? 1 : most < want ? most : want);
        chunk_rows = (rows + splits - 1) / splits;
    }
};

template <class T>
void launch_backward(const wc_act8_args& a, cudaStream_t s) {
    const bool units = a.width % 8 == 0 && aligned(a.x, a.ld_x, sizeof(T)) && aligned(a.out, a.ld_out, sizeof(T));
    const Shape g(a.rows, a.width, units);
    float* part = a.dbias ? static_cast<float*>(a.workspace) : nullptr;
    const dim3 grid(g.tiles, g.splits);
    if (units) k_gelu8_backward<T, true><<<grid, THREADS, 0, s>>>(a, g.blocks, g.lanes, g.chunk_rows, part);
    else k_gelu8_backward<T, false><<<grid, THREADS, 0, s>>>(a, g.blocks, g.lanes, g.chunk_rows, part);
    if (part) launch_colsum<float>(part, g.splits, a.width, a.width, a.dbias, s);
}

}  // namespace

void launch_act8_pack(const wc_act8_args& a, cudaStream_t s) { launch_type<PACK>(a, s); }
void launch_act8_unpack(const wc_act8_args& a, cudaStream_t s) { launch_type<UNPACK>(a, s); }
void launch_gelu8(const wc_act8_args& a, cudaStream_t s) { launch_type<GELU>(a, s); }
uint64_t gelu8_workspace(int64_t rows, int64_t width) {
    if (!width) return 0;
    const Shape one(rows, width, false);
    const int splits = width % 8 ? one.splits : std::max(one.splits, Shape(rows, width, true).splits);
    return (uint64_t)splits * width * sizeof(float);
}
void launch_gelu8_backward(const wc_act8_args& a, cudaStream_t s) {
    if (a.type == WC_F32) launch_backward<float>(a, s);
    else if (a.type == WC_F16) launch_backward<__half>(a, s);
    else launch_backward<__nv_bfloat16>(a, s);
}

}  // namespace wctrain
