// Activations in 8 bits: blocks of 32 values along a row share a power-of-two
// unit (train.cuh act8_code), so a stored value is a whole number times that
// unit and is exact in bf16.
//
// All of these move few bytes a value, and what comes first is the instructions:
// at 30 to 55 a value (measured, of earlier forms) the SMs issue for longer than
// the memory takes. So arithmetic is on pairs, index divisions are products, and
// what is a block's alone is computed once for it. Where addresses and strides
// allow, a thread holds 8 consecutive values (16 bytes of a 16-bit type in one
// load, 8 bytes of q in one store) and 4 threads a block: the largest magnitude
// takes two shuffles. Elsewhere a warp holds 8 blocks, one value of each a
// thread, so that its loads and stores are still next to each other.
//
// On a B200 131071 x 897 in f32 is packed and read back in 228 to 241 us (4.9 to 5.2
// TB/s of the 6.5 that a copy reaches), 131072 x 1024 in bf16 in 143 us (5.7 TB/s);
// GELU forward and backward of 4095 x 16384 in bf16 takes 139 to 143 us (4.7 to 4.9
// TB/s).
#include <algorithm>
#include <type_traits>

#include "colsum.cuh"

namespace wctrain {

namespace {

constexpr int THREADS = 256;

// 8 values of a row from column c on; those past the width (a whole number of 8s) are 0
template <class T>
struct Raw {
    alignas(16) uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p, bool in) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = in ? __ldcs(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(Pair* v) const {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = umma::f2(u[2 * i], u[2 * i + 1]);
            else if constexpr (std::is_same<T, __nv_bfloat16>::value) v[i] = umma::f2(u[i] << 16, u[i] & 0xffff0000u);
            else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
                v[i] = umma::f2(f.x, f.y);
            }
        }
    }
};
template <class T>
__device__ __forceinline__ void store8(T* p, const Pair* v) {
    alignas(16) uint32_t u[2 * sizeof(T)];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float lo = umma::f2_lo(v[i]), hi = umma::f2_hi(v[i]);
        if constexpr (sizeof(T) == 4) u[2 * i] = __float_as_uint(lo), u[2 * i + 1] = __float_as_uint(hi);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(&u[i]) = __floats2bfloat162_rn(lo, hi);
        else *reinterpret_cast<__half2*>(&u[i]) = __floats2half2_rn(lo, hi);
    }
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, reinterpret_cast<const uint4*>(u)[i]);
}
__device__ __forceinline__ void load_bias8(const float* p, Pair* v) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = umma::f2(a.x, a.y), v[1] = umma::f2(a.z, a.w), v[2] = umma::f2(b.x, b.y), v[3] = umma::f2(b.z, b.w);
}

// i / d for i < 2^31 by a product with floor(2^32 / d), which gives the quotient or one less
struct Divisor {
    uint32_t d, m;
    explicit Divisor(uint32_t v) : d(v), m(v > 1 ? (uint32_t)((1ull << 32) / v) : 0xffffffffu) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t i, uint32_t* rest) const {
        uint32_t q = __umulhi(i, m), r = i - q * d;
        if (r >= d) ++q, r -= d;
        *rest = r;
        return q;
    }
};

enum { PACK, UNPACK, GELU };

template <class T, int WHAT>
__global__ void __launch_bounds__(THREADS) k_act8(wc_act8_args a, Divisor chunks, uint32_t total) {
    const uint32_t i = blockIdx.x * THREADS + threadIdx.x;
    const bool in = i < total;  // total is a multiple of 4: a block's threads are in or out together
    uint32_t chunk;
    const uint32_t row = chunks(in ? i : 0, &chunk);
    const int64_t c = (int64_t)chunk * 8;
    const bool here = in && c < a.width;
    Pair v[4];
    if constexpr (WHAT == UNPACK) {
        if (!here) return;
        dequantise8(__ldcs(reinterpret_cast<const uint2*>(a.q) + i), a.scale[i >> 2], v);
        store8(static_cast<T*>(a.out) + row * a.ld_out + c, v);
    } else {
        Raw<T> x;
        x.load(static_cast<const T*>(a.x) + row * a.ld_x + c, here);
        x.get(v);
        if constexpr (WHAT == GELU) {
            if (here) {
                if (a.bias) {
                    Pair b[4];
                    load_bias8(a.bias + c, b);
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = add(v[k], b[k]);
                }
                Pair y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = gelu(v[k]);
                store8(static_cast<T*>(a.out) + row * a.ld_out + c, y);
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

// The same, a warp 8 blocks, a column of each a lane; lane k keeps what is the k-th block's. FLAT: 8 next to each other in
// the matrix, which end in a later row than they begin in (`units` is a row's blocks); else a run of a row's (`units` is a
// row's runs), whose addresses are known from the first.
template <class T, int WHAT, bool FLAT>
__global__ void __launch_bounds__(THREADS) k_act8_runs(wc_act8_args a, int blocks, Divisor units, uint32_t total) {
    const uint32_t i = (blockIdx.x * THREADS + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    if (FLAT ? i * 8 >= total : i >= total) return;
    // this lane's block of the eight, and the place of the first one's q and scale
    uint32_t run;
    const uint32_t mine = FLAT ? min(i * 8 + (lane & 7), total - 1) : i, line = units(mine, &run);
    const int64_t b0 = FLAT ? (int64_t)i * 8 : (int64_t)line * blocks + run * 8;
    const int left = FLAT ? (int)(total - i * 8) : blocks - (int)run * 8;
    int8_t* q = a.q + b0 * 32 + lane;
    uint8_t* scale = a.scale + b0;
    // the k-th block's first column, how many are left in its row from this lane's on, and that one's address
    auto first = [&](int k) { return FLAT ? __shfl_sync(0xffffffffu, run, k) * 32 : run * 256 + k * 32; };
    auto cols = [&](int k) {
        const uint32_t c = first(k);
        return k < left ? (int)(a.width - c) - (int)lane : 0;
    };
    auto at = [&](auto* base, int64_t ld, int k) {
        if constexpr (FLAT) return base + __shfl_sync(0xffffffffu, line, k) * ld + first(k) + lane;
        else return base + (line * ld + run * 256 + lane) + k * 32;
    };
    const T* x = static_cast<const T*>(a.x);
    T* out = static_cast<T*>(a.out);
    if constexpr (WHAT == UNPACK) {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = k < left ? (uint32_t)(uint8_t)__ldcs(q + k * 32) : 0;
        const float unit = act8_unit((int)lane < min(left, 8) ? scale[lane] : 1);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float v = act8_number(w[k]) * __shfl_sync(0xffffffffu, unit, k);
            T* to = at(out, a.ld_out, k);
            if (cols(k) > 0) __stcs(to, from_f<T>(v));
        }
    } else {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const T* from = at(x, a.ld_x, k);
            v[k] = cols(k) > 0 ? to_f(__ldcs(from)) : 0.0f;
        }
        if constexpr (WHAT == GELU)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                T* to = at(out, a.ld_out, k);
                const uint32_t c = first(k) + lane;
                if (cols(k) > 0) {
                    if (a.bias) v[k] += a.bias[c];
                    __stcs(to, from_f<T>(gelu(v[k])));
                }
            }
        // magnitudes are compared as integers, where NaN is above infinity above the rest, so either shows in the code
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(v[k]) & 0x7fffffffu);
            if (lane == k) top = m;
        }
        const uint32_t code = act8_code(__uint_as_float(top));
        if ((int)lane < min(left, 8)) scale[lane] = (uint8_t)code;
        if (__any_sync(0xffffffffu, code >= ACT8_LARGEST)) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t its = __shfl_sync(0xffffffffu, code, k);
                if (k < left) q[k * 32] = act8_whole(v[k], its);
            }
        } else {
            const float inv = act8_inverse(code);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float its = __shfl_sync(0xffffffffu, inv, k);
                if (k < left) q[k * 32] = (int8_t)__float_as_uint(fmaf(v[k], its, 12582912.0f));
            }
        }
    }
}

// dz = da GELU'(z8). The CTA's threads keep their columns and walk down the
// rows [blockIdx.y * chunk_rows, ...): `lanes` threads a row, each 8 columns.
// K = 0: consecutive ones. Else `lanes` is a number of warps times 32, and a
// warp has 32 K columns, thread by thread next to each other.
template <class T, int K>
__global__ void __launch_bounds__(THREADS) k_gelu8_backward(wc_act8_args a, int blocks, int lanes, int64_t chunk_rows, float* part) {
    constexpr bool UNITS = K == 0;
    constexpr int EACH = UNITS ? 8 : K;  // columns of a thread
    __shared__ float s[THREADS][9];
    const int per = THREADS / lanes, r = threadIdx.x / lanes, at = blockIdx.x * lanes + threadIdx.x % lanes;
    const int step = UNITS ? 1 : 32, c = UNITS ? at * 8 : (at & ~31) * K + (at & 31);
    const bool in = r < per && c < a.width;
    const int64_t first = blockIdx.y * chunk_rows, last = min(first + chunk_rows, a.rows);
    Pair acc[4] = {0, 0, 0, 0};  // (pairs of zeros)
    if constexpr (UNITS) {
        if (in) {
            const int64_t row_q = (int64_t)blocks * 32;
            const T* x = static_cast<const T*>(a.x) + (first + r) * a.ld_x + c;
            T* out = static_cast<T*>(a.out) + (first + r) * a.ld_out + c;
            const int8_t* q = a.q + (first + r) * row_q + c;
            const uint8_t* scale = a.scale + (first + r) * blocks + c / 32;
            Raw<T> d;
            uint2 w = make_uint2(0, 0);
            uint32_t code = 1;
            auto fetch = [&](int64_t t) {
                if (t >= last) return;
                d.load(x, true), w = __ldcs(reinterpret_cast<const uint2*>(q)), code = *scale;
                x += per * a.ld_x, q += per * row_q, scale += per * blocks;
            };
            fetch(first + r);
            for (int64_t t = first + r; t < last; t += per) {
                Pair z[4], g[4];
                d.get(g), dequantise8(w, code, z), gelu_cut(code, z, 4);
                fetch(t + per);
#pragma unroll
                for (int k = 0; k < 4; ++k) g[k] = mul(g[k], gelu_slope(z[k])), acc[k] = add(acc[k], g[k]);
                store8(out, g);
                out += per * a.ld_out;
            }
        }
    } else if (in) {
        for (int64_t t = first + r; t < last; t += per) {
            const T* x = static_cast<const T*>(a.x) + t * a.ld_x + c;
            T* out = static_cast<T*>(a.out) + t * a.ld_out + c;
            const int8_t* q = a.q + t * blocks * 32 + c;
            const uint8_t* scale = a.scale + t * blocks + c / 32;
            const int left = (int)(a.width - c);
            float d[8] = {};
            uint32_t w[8], code[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool here = k < K && k * 32 < left;
                d[k] = here ? to_f(__ldcs(x + k * 32)) : 0.0f, w[k] = here ? (uint32_t)(uint8_t)__ldcs(q + k * 32) : 0, code[k] = here ? scale[k] : 1;
            }
#pragma unroll
            for (int k = 0; 2 * k < K; ++k) {
                Pair z = mul(umma::f2(act8_number(w[2 * k]), act8_number(w[2 * k + 1])), umma::f2(act8_unit(code[2 * k]), act8_unit(code[2 * k + 1])));
                if (max(code[2 * k], code[2 * k + 1]) > 147) {
                    Pair lo = umma::f2(umma::f2_lo(z), 0.0f), hi = umma::f2(umma::f2_hi(z), 0.0f);
                    gelu_cut(code[2 * k], &lo, 1), gelu_cut(code[2 * k + 1], &hi, 1);
                    z = umma::f2(umma::f2_lo(lo), umma::f2_lo(hi));
                }
                const Pair g = mul(umma::f2(d[2 * k], d[2 * k + 1]), gelu_slope(z));
                acc[k] = add(acc[k], g);
                if (2 * k * 32 < left) __stcs(out + 2 * k * 32, from_f<T>(umma::f2_lo(g)));
                if (2 * k + 1 < K && (2 * k + 1) * 32 < left) __stcs(out + (2 * k + 1) * 32, from_f<T>(umma::f2_hi(g)));
            }
        }
    }
    if (!part) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) s[threadIdx.x][k] = k & 1 ? umma::f2_hi(acc[k / 2]) : umma::f2_lo(acc[k / 2]);
    __syncthreads();
    if (in && r == 0)
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            float v = s[threadIdx.x][k];
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
                           (WHAT == PACK || aligned(b.out, a.ld_out, sizeof(T))) && ((uintptr_t)a.bias & 15) == 0;
        if (units) {
            const uint32_t total = (uint32_t)(b.rows * chunks);
            k_act8<T, WHAT><<<(total + THREADS - 1) / THREADS, THREADS, 0, s>>>(b, Divisor((uint32_t)chunks), total);
        } else {
            // Runs of a row unless most of one is past it (1000000 x 31 in bf16 packs in 39 us, in runs with one block of
            // eight it took 178; 100000 x 333, with 11 blocks of 16, in 44 us in runs, 47 without)
            const uint32_t blocks = (uint32_t)(chunks / 4), runs = (blocks + 7) / 8;
            if (blocks < 4) {
                const uint32_t total = (uint32_t)(b.rows * blocks), warps = (total + 7) / 8;
                k_act8_runs<T, WHAT, true><<<(warps + 7) / 8, THREADS, 0, s>>>(b, (int)blocks, Divisor(blocks), total);
            } else {
                const uint32_t total = (uint32_t)(b.rows * runs);
                k_act8_runs<T, WHAT, false><<<(unsigned)((total + 7ull) / 8), THREADS, 0, s>>>(b, (int)blocks, Divisor(runs), total);
            }
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
    int each = 8;  // columns of a thread
    Shape(int64_t rows, int64_t width, bool units) {
        blocks = (int)((width + 31) / 32);
        // without units: the most columns a thread with little past the width (an eighth), else a warp's 32
        const auto past = [&](int k) { return (blocks + k - 1) / k * k - blocks; };
        if (!units)
            while (each > 1 && past(each) * 8 > blocks) each /= 2;
        const int threads = units ? (int)(width / 8) : (blocks + each - 1) / each * 32, whole = units ? 1 : 32;
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
    const auto kernel = units ? k_gelu8_backward<T, 0>
                        : g.each == 8 ? k_gelu8_backward<T, 8>
                        : g.each == 4 ? k_gelu8_backward<T, 4>
                        : g.each == 2 ? k_gelu8_backward<T, 2>
                                      : k_gelu8_backward<T, 1>;
    kernel<<<grid, THREADS, 0, s>>>(a, g.blocks, g.lanes, g.chunk_rows, part);
    if (part) launch_colsum(part, g.splits, a.width, a.width, 1, ColSums{{a.dbias}}, s);
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
